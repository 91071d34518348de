"""Python bindings (ctypes) for the token mixers of librl_sampler.so
(include/rl_mixers.h): rotary positions, the paged key-value cache, attention of
new tokens over it, by themselves or behind shared prefixes, the gated delta rule, the
short causal convolution and the selective state space scan.

As in rl_sampler.py this only marshals arguments: tensors are torch tensors on the
handle's device, [rows][heads][dim] with the last axis contiguous and any strides
before it, calls go to the current stream unless one is given, and a refusal of
the library raises rl_sampler.SamplerError. Every tensor is checked before the
call: a kernel given an address of the host or of another device would fault.
"""
import ctypes
import struct

import torch

import rl_sampler
from rl_sampler import _check, _u32, _u64, _vp

TYPES = {"f32": 0, "f16": 1, "bf16": 2, "i8": 3, "f8": 4}
LAYOUTS = {"half": 0, "interleaved": 1}
ACTIVATIONS = {"none": 0, "silu": 1}
SCALINGS = {"none": 0, "linear": 1, "ntk": 2, "yarn": 3}

_HEADS = struct.Struct("=QQQIIII")  # rl_heads
_pack = _HEADS.pack
_i32, _f32 = ctypes.c_int, ctypes.c_float
_bound = None


class RotarySpec(ctypes.Structure):
    """rl_rotary_spec."""

    _fields_ = [("dims", _u32), ("layout", _u32), ("scaling", _u32), ("original", _u32),
                ("base", ctypes.c_double), ("factor", ctypes.c_double), ("beta_fast", ctypes.c_double),
                ("beta_slow", ctypes.c_double), ("magnitude", ctypes.c_double)]


def lib():
    """The library with this header's signatures declared."""
    global _bound
    if _bound is None:
        L = rl_sampler.lib()
        out = ctypes.POINTER(_vp)
        heads = ctypes.c_char_p  # packed rl_heads
        L.rl_rotary_create.argtypes = [_i32, ctypes.POINTER(RotarySpec), out]
        L.rl_rotary_frequencies.argtypes = [_vp, ctypes.POINTER(ctypes.c_double), ctypes.POINTER(ctypes.c_double)]
        L.rl_rotary_rows.argtypes = [_vp, _vp, _u32, heads, heads, _u32, _i32, _vp]
        L.rl_kv_cache_create.argtypes = [_i32, _u32, _u32, _u32, _u32, _u32, out]
        L.rl_kv_cache_bytes.argtypes = [_vp]
        L.rl_kv_cache_bytes.restype = _u64
        L.rl_kv_cache_write.argtypes = [_vp, heads, heads, _vp, _u32, _vp, _vp, _vp]
        L.rl_kv_cache_read.argtypes = [_vp, _vp, _u32, heads, heads, _vp]
        L.rl_attention_create.argtypes = [_i32, _u32, _u32, _u32, _u32, _u32, out]
        L.rl_attention_rows.argtypes = [_vp, _vp, heads, heads, _vp, _u32, _vp, _vp, _u32, _vp, _u32, _f32, _u32, _u32,
                                        _u32, _vp]
        L.rl_delta_create.argtypes = [_i32, _u32, _u32, _u32, _u32, _u32, _u32, out]
        L.rl_delta_rows.argtypes = [_vp, heads, heads, heads, heads, _vp, _u64, _vp, _u64, _vp, _u64, _vp, _vp, _vp,
                                    _u32, _u32, _f32, _f32, _u32, _vp]
        L.rl_attention_shared.argtypes = [_vp, _vp, heads, heads, _vp, _u32, _vp, _vp, _u32, _vp, _u32, _vp, _vp, _u32,
                                          _vp, _u32, _f32, _u32, _u32, _u32, _vp]
        L.rl_conv_create.argtypes = [_i32, _u32, _u32, _vp, _vp, _u32, out]
        L.rl_conv_rows.argtypes = [_vp, heads, heads, _vp, _u64, _vp, _vp, _vp, _u32, _u32, _vp]
        L.rl_scan_create.argtypes = [_i32, _u32, _u32, _u32, _u32, _u32, _vp, _vp, _vp, out]
        L.rl_scan_rows.argtypes = [_vp, heads, heads, heads, heads, heads, heads, _vp, _u64, _vp, _vp, _vp, _u32, _u32,
                                   _i32, _u32, _vp]
        for name in ("rl_rotary_destroy", "rl_kv_cache_destroy", "rl_attention_destroy", "rl_delta_destroy",
                     "rl_conv_destroy", "rl_scan_destroy"):
            f = getattr(L, name)
            f.argtypes, f.restype = [_vp], None
        _bound = L
    return _bound


_codes = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


def _elsewhere(t, device):
    """The refusal of a tensor that is not on the handle's device. (The comparisons
    stand in line: each costs a call a twentieth of a microsecond as it is.)"""
    return ValueError("the tensors of a call are on the handle's device, cuda:%d, not %s" % (device, t.device))


def _stream(device, stream):
    """The stream given, or the device's current one (without the Stream object of
    torch.cuda.current_stream, which costs 3 us a call)."""
    return torch._C._cuda_getCurrentRawStream(device) if stream is None else stream


def _heads(t, device=None):
    """A tensor [rows][heads][dim] as a packed rl_heads; on the device, if one is
    named."""
    if device is not None and t.get_device() != device:
        raise _elsewhere(t, device)
    _, heads, dim = t.shape
    rows, per, one = t.stride()
    if one != 1 or t.dtype not in _codes:
        raise ValueError("a tensor of f32, f16 or bf16 whose last axis is contiguous")
    return _pack(t.data_ptr(), rows, per, heads, dim, _codes[t.dtype], 0)


def _channels(t, device):
    """A tensor [rows][channels] as a packed rl_heads of one head."""
    if t.get_device() != device:
        raise _elsewhere(t, device)
    _, channels = t.shape
    rows, one = t.stride()
    if (one != 1 and channels > 1) or t.dtype not in _codes:
        raise ValueError("a tensor of f32, f16 or bf16 whose last axis is contiguous")
    return _pack(t.data_ptr(), rows, 0, 1, channels, _codes[t.dtype], 0)


def _states(states, dtype, shape, device):
    """The address of a pool of states."""
    if states.get_device() != device:
        raise _elsewhere(states, device)
    if states.dtype != dtype or not states.is_contiguous() or states.shape[1:] != shape:
        raise ValueError("states are contiguous %s [slots]%s" % (dtype, list(shape)))
    return states.data_ptr()


def _host(t, shape):
    """A contiguous f32 copy of weights on the host, or None."""
    if t is None:
        return None
    if t.shape != shape:
        raise ValueError("weights of another shape than %s" % list(shape))
    return t.detach().to("cpu", torch.float32).contiguous()


def _at(t):
    return None if t is None else t.data_ptr()


def _index(t, dtype, count, device):
    """The address of a contiguous index tensor of at least `count` values."""
    if t.get_device() != device:
        raise _elsewhere(t, device)
    if t.dtype != dtype or not t.is_contiguous() or t.numel() < count:
        raise ValueError("a contiguous %s tensor of %d values" % (dtype, count))
    return t.data_ptr()


class _Handle:
    _destroy = None
    device = 0

    def close(self):
        if getattr(self, "h", None):
            getattr(lib(), self._destroy)(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class DeviceRotary(_Handle):
    """rl_rotary_create / rl_rotary_rows: rotary positions of the first `dims`
    values of a head."""

    _destroy = "rl_rotary_destroy"

    def __init__(self, dims, base=10000.0, layout="half", scaling="none", factor=1.0, original=0, beta_fast=0.0,
                 beta_slow=0.0, magnitude=0.0, device=0):
        spec = RotarySpec(dims, LAYOUTS[layout], SCALINGS[scaling], original, base, factor, beta_fast, beta_slow,
                          magnitude)
        h = _vp()
        _check(lib().rl_rotary_create(device, ctypes.byref(spec), ctypes.byref(h)))
        self.h, self.dims, self.device = h, dims, device

    def frequencies(self):
        """(radians a position of every pair, the magnitude)."""
        radians, magnitude = (ctypes.c_double * (self.dims // 2))(), ctypes.c_double()
        _check(lib().rl_rotary_frequencies(self.h, radians, ctypes.byref(magnitude)))
        return list(radians), magnitude.value

    def apply(self, x, positions, out=None, second=None, second_out=None, inverse=False, stream=None):
        """Turns x [rows][heads][dim] by positions [rows] (int64) into `out` (x
        itself if None), and `second` likewise in the same launch."""
        rows, device = x.shape[0], self.device
        out = x if out is None else out
        ins, outs, tensors = _heads(x, device), _heads(out, device), 1
        if out.shape != x.shape:
            raise ValueError("out has another shape")
        if second is not None:
            second_out = second if second_out is None else second_out
            if second.shape[0] != rows or second_out.shape != second.shape:
                raise ValueError("the second tensor has other rows, or its output another shape")
            ins, outs, tensors = ins + _heads(second, device), outs + _heads(second_out, device), 2
        _check(lib().rl_rotary_rows(self.h, _index(positions, torch.int64, rows, device), rows, ins, outs, tensors,
                                    int(inverse), _stream(device, stream)))


class DeviceCache(_Handle):
    """rl_kv_cache_create / _write / _read: one layer's paged keys and values, in
    f16, bf16, or quantised to i8 or f8 (e4m3) as they are written."""

    _destroy = "rl_kv_cache_destroy"

    def __init__(self, pages, page, kv_heads, dim, format="bf16", device=0):
        h = _vp()
        _check(lib().rl_kv_cache_create(device, pages, page, kv_heads, dim, TYPES[format], ctypes.byref(h)))
        self.h, self.device = h, device
        self.pages, self.page, self.kv_heads, self.dim, self.format = pages, page, kv_heads, dim, format

    def bytes(self):
        return lib().rl_kv_cache_bytes(self.h)

    def write(self, keys, values, slots, rotary=None, positions=None, stream=None):
        """Rows keys[i], values[i] to slots[i] (int64; negative: left out, the others
        distinct), the keys turned by positions[i] first if a DeviceRotary is given."""
        rows, device = keys.shape[0], self.device
        if values.shape[0] != rows:
            raise ValueError("keys and values have one row a slot")
        at = None if rotary is None else _index(positions, torch.int64, rows, device)
        _check(lib().rl_kv_cache_write(self.h, _heads(keys, device), _heads(values, device),
                                       _index(slots, torch.int64, rows, device), rows,
                                       None if rotary is None else rotary.h, at, _stream(device, stream)))

    def read(self, slots, keys, values, stream=None):
        """Into keys[i], values[i] what slots[i] holds (NaN outside the cache)."""
        rows, device = keys.shape[0], self.device
        if values.shape[0] != rows:
            raise ValueError("keys and values have one row a slot")
        _check(lib().rl_kv_cache_read(self.h, _index(slots, torch.int64, rows, device), rows, _heads(keys, device),
                                      _heads(values, device), _stream(device, stream)))


class DeviceAttention(_Handle):
    """rl_attention_create / rl_attention_rows: attention of new tokens over a
    DeviceCache."""

    _destroy = "rl_attention_destroy"

    def __init__(self, max_rows, q_heads, kv_heads, dim, max_len, device=0):
        h = _vp()
        _check(lib().rl_attention_create(device, max_rows, q_heads, kv_heads, dim, max_len, ctypes.byref(h)))
        self.h, self.q_heads, self.scale, self.device = h, q_heads, dim ** -0.5, device

    def rows(self, cache, q, out, lens, pages, starts=None, lse=None, scale=None, window=0, most_rows=0, max_len=0,
             stream=None):
        """q, out [rows][q_heads][dim]; lens int32 [seqs]; pages int32
        [seqs][width]; starts int32 [seqs + 1] (None: one row a sequence); lse f32
        [rows][q_heads] if wanted; scale: dim^-1/2 if None."""
        rows, seqs, width, device = q.shape[0], pages.shape[0], pages.shape[1], self.device
        if out.shape != q.shape:
            raise ValueError("out has another shape than q")
        _check(lib().rl_attention_rows(
            self.h, cache.h, _heads(q, device), _heads(out, device),
            None if lse is None else _index(lse, torch.float32, rows * self.q_heads, device), rows,
            None if starts is None else _index(starts, torch.int32, seqs + 1, device),
            _index(lens, torch.int32, seqs, device), seqs, _index(pages, torch.int32, seqs * width, device), width,
            self.scale if scale is None else scale, window, most_rows, max_len, _stream(device, stream)))


    def shared(self, cache, q, out, lens, pages, groups, prefix_lens, prefix_pages, starts=None, lse=None, scale=None,
               most_rows=0, max_len=0, max_prefix=0, stream=None):
        """As rows(), where the sequences groups[g] .. groups[g + 1] (int32
        [prefixes + 1]) have the prefix_lens[g] (int32) tokens of prefix_pages[g] (int32
        [prefixes][width]) before their own: lens and pages are of their own tokens."""
        rows, seqs, width, device = q.shape[0], pages.shape[0], pages.shape[1], self.device
        count, wide = prefix_pages.shape
        if out.shape != q.shape:
            raise ValueError("out has another shape than q")
        _check(lib().rl_attention_shared(
            self.h, cache.h, _heads(q, device), _heads(out, device),
            None if lse is None else _index(lse, torch.float32, rows * self.q_heads, device), rows,
            None if starts is None else _index(starts, torch.int32, seqs + 1, device),
            _index(lens, torch.int32, seqs, device), seqs, _index(pages, torch.int32, seqs * width, device), width,
            _index(groups, torch.int32, count + 1, device), _index(prefix_lens, torch.int32, count, device), count,
            _index(prefix_pages, torch.int32, count * wide, device), wide, self.scale if scale is None else scale,
            most_rows, max_len, max_prefix, _stream(device, stream)))


class DeviceDelta(_Handle):
    """rl_delta_create / rl_delta_rows: the gated delta rule over a pool of f32
    states."""

    _destroy = "rl_delta_destroy"

    def __init__(self, max_rows, max_seqs, key_heads, value_heads, key_dim, value_dim, device=0):
        h = _vp()
        _check(lib().rl_delta_create(device, max_rows, max_seqs, key_heads, value_heads, key_dim, value_dim,
                                     ctypes.byref(h)))
        self.h, self.scale, self.device = h, key_dim ** -0.5, device
        self.state = (value_heads, key_dim, value_dim)

    def rows(self, q, k, v, g, beta, out, states, slots_in, slots_out, starts=None, scale=None, normalise=False,
             eps=1e-6, most_rows=0, stream=None):
        """q, k [rows][key_heads][key_dim]; v, out [rows][value_heads][value_dim];
        g, beta f32 [rows][value_heads]; states f32 [slots][value_heads][key_dim]
        [value_dim], contiguous; slots_in, slots_out int32 [seqs] (negative: none;
        the slots written distinct); starts int32 [seqs + 1] (None: one row a
        sequence); scale: key_dim^-1/2 if None."""
        rows, seqs, device = q.shape[0], slots_in.shape[0], self.device
        if k.shape[0] != rows or v.shape[0] != rows or out.shape[0] != rows:
            raise ValueError("q, k, v and out have one row a token")
        for x in (g, beta, states):
            if x.get_device() != device:
                raise _elsewhere(x, device)
        for x in (g, beta):
            # One head has no next one: its stride says nothing.
            if x.dtype != torch.float32 or x.shape != (rows, self.state[0]) or (x.stride(1) != 1 and x.shape[1] > 1):
                raise ValueError("g and beta are f32 [rows][value_heads], heads contiguous")
        if states.dtype != torch.float32 or not states.is_contiguous() or states.shape[1:] != self.state:
            raise ValueError("states are contiguous f32 [slots][value_heads][key_dim][value_dim]")
        _check(lib().rl_delta_rows(
            self.h, _heads(q, device), _heads(k, device), _heads(v, device), _heads(out, device), g.data_ptr(),
            g.stride(0), beta.data_ptr(), beta.stride(0), states.data_ptr(), states.shape[0],
            _index(slots_in, torch.int32, seqs, device), _index(slots_out, torch.int32, seqs, device),
            None if starts is None else _index(starts, torch.int32, seqs + 1, device), rows, seqs,
            self.scale if scale is None else scale, eps if normalise else -1.0, most_rows, _stream(device, stream)))


class DeviceConv(_Handle):
    """rl_conv_create / rl_conv_rows: the short causal convolution of every channel,
    over a pool of states."""

    _destroy = "rl_conv_destroy"

    def __init__(self, weight, bias=None, activation="silu", device=0):
        """weight [channels][width], bias [channels] if any: copied."""
        channels, width = weight.shape
        w, b, h = _host(weight, weight.shape), _host(bias, (channels,)), _vp()
        _check(lib().rl_conv_create(device, channels, width, w.data_ptr(), _at(b), ACTIVATIONS[activation],
                                    ctypes.byref(h)))
        self.h, self.device, self.state = h, device, (width - 1, channels)

    def rows(self, x, out, states, slots_in, slots_out, starts=None, stream=None):
        """x, out [rows][channels]; states [slots][width - 1][channels] of x's type,
        contiguous; slots_in, slots_out int32 [seqs] (negative: none; the slots written
        distinct); starts int32 [seqs + 1] (None: one row a sequence)."""
        rows, seqs, device = x.shape[0], slots_in.shape[0], self.device
        if out.shape != x.shape:
            raise ValueError("out has another shape than x")
        _check(lib().rl_conv_rows(
            self.h, _channels(x, device), _channels(out, device), _states(states, x.dtype, self.state, device),
            states.shape[0], _index(slots_in, torch.int32, seqs, device), _index(slots_out, torch.int32, seqs, device),
            None if starts is None else _index(starts, torch.int32, seqs + 1, device), rows, seqs,
            _stream(device, stream)))


class DeviceScan(_Handle):
    """rl_scan_create / rl_scan_rows: the selective state space scan over a pool of f32
    states."""

    _destroy = "rl_scan_destroy"

    def __init__(self, max_rows, max_seqs, a, groups=1, skip=None, dt_bias=None, device=0):
        """a [channels][state_dim], skip and dt_bias [channels] if any: copied."""
        channels, state = a.shape
        decay, d, bias, h = _host(a, a.shape), _host(skip, (channels,)), _host(dt_bias, (channels,)), _vp()
        _check(lib().rl_scan_create(device, max_rows, max_seqs, channels, groups, state, decay.data_ptr(), _at(d),
                                    _at(bias), ctypes.byref(h)))
        self.h, self.device, self.state = h, device, (channels, state)

    def rows(self, x, dt, b, c, out, states, slots_in, slots_out, starts=None, z=None, softplus=True, most_rows=0,
             stream=None):
        """x, dt, out and z (if any) [rows][channels]; b, c [rows][groups][state_dim];
        states f32 [slots][channels][state_dim], contiguous; slots_in, slots_out int32
        [seqs] (negative: none; the slots written distinct); starts int32 [seqs + 1]
        (None: one row a sequence)."""
        rows, seqs, device = x.shape[0], slots_in.shape[0], self.device
        for t in (dt, b, c, out):
            if t.shape[0] != rows:
                raise ValueError("the tensors of a call have one row a token")
        if z is not None and z.shape[0] != rows:
            raise ValueError("the tensors of a call have one row a token")
        _check(lib().rl_scan_rows(
            self.h, _channels(x, device), _channels(dt, device), None if z is None else _channels(z, device),
            _heads(b, device), _heads(c, device), _channels(out, device),
            _states(states, torch.float32, self.state, device), states.shape[0],
            _index(slots_in, torch.int32, seqs, device), _index(slots_out, torch.int32, seqs, device),
            None if starts is None else _index(starts, torch.int32, seqs + 1, device), rows, seqs, int(softplus),
            most_rows, _stream(device, stream)))
