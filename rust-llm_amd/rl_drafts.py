"""Python binding (ctypes) of the verification of drafted tokens in librl_sampler.so
(include/rl_drafts.h).

As in rl_mixers.py this only marshals arguments: tensors are torch tensors on the
handle's device, calls go to the current stream unless one is given, and a refusal of
the library raises rl_sampler.SamplerError.
"""
import ctypes
import struct

import torch

import rl_sampler
from rl_mixers import _Handle, _elsewhere, _index, _stream
from rl_sampler import _check, _u32, _vp

_PROBS = struct.Struct("=QQQQ")  # rl_probs
_bound = None


def lib():
    """The library with this header's signatures declared."""
    global _bound
    if _bound is None:
        L = rl_sampler.lib()
        probs = ctypes.c_char_p  # packed rl_probs
        L.rl_drafts_create.argtypes = [ctypes.c_int, _u32, _u32, ctypes.POINTER(_vp)]
        L.rl_drafts_destroy.argtypes, L.rl_drafts_destroy.restype = [_vp], None
        L.rl_drafts_verify.argtypes = [_vp, probs, probs, _vp, _vp, _vp, _vp, _u32, _u32, _vp, _vp, _vp]
        _bound = L
    return _bound


def _probs(p, ids, kept, rows, vocab, device):
    """Rows of probabilities as a packed rl_probs."""
    if p.get_device() != device:
        raise _elsewhere(p, device)
    if p.dtype != torch.float32 or p.dim() != 2 or p.shape[0] < rows or (p.stride(1) != 1 and p.shape[1] > 1 and p.shape[0]):
        raise ValueError("probabilities are f32 [%d rows or more][..], the last axis contiguous" % rows)
    stride = p.stride(0) if p.shape[0] > 1 else max(p.stride(0), p.shape[1])
    if (ids is None) != (kept is None):
        raise ValueError("a list has ids and kept counts")
    if ids is None:
        if p.shape[1] != vocab:
            raise ValueError("rows of probabilities have the handle's %d tokens" % vocab)
        return _PROBS.pack(p.data_ptr(), stride, 0, 0)
    if ids.get_device() != device:
        raise _elsewhere(ids, device)
    if ids.dtype != torch.int32 or ids.shape != p.shape or not ids.is_contiguous() or not p.is_contiguous():
        raise ValueError("ids are int32 of the probabilities' shape, both contiguous")
    return _PROBS.pack(p.data_ptr(), p.shape[1], ids.data_ptr(), _index(kept, torch.int32, rows, device))


class DeviceDrafts(_Handle):
    """rl_drafts_create / rl_drafts_verify: how many drafted tokens the target's
    probabilities accept, and the token after them."""

    _destroy = "rl_drafts_destroy"

    def __init__(self, max_seqs, vocab, device=0):
        h = _vp()
        _check(lib().rl_drafts_create(device, max_seqs, vocab, ctypes.byref(h)))
        self.h, self.device, self.vocab = h, device, vocab

    def verify(self, target, drafted, starts, uniforms, draws, accepted, tokens, draft=None, target_ids=None,
               target_kept=None, draft_ids=None, draft_kept=None, stream=None):
        """drafted int32 [drafts], sequence s's from starts[s] on (int32 [seqs + 1]);
        target f32 [drafts + seqs][vocab], a sequence's rows one more than its drafts;
        draft f32 [drafts][vocab] (None: the drafts were not drawn). With ids (int32) and
        kept (int32 [rows]) both are the candidate lists of sample_rows instead.
        uniforms f32 [drafts], draws f32 [seqs]; accepted int32 [seqs] and tokens int32
        [drafts + seqs] are written."""
        drafts, seqs, device = drafted.shape[0], draws.shape[0], self.device
        if starts.numel() != seqs + 1 or tokens.numel() != drafts + seqs:
            raise ValueError("starts has one more and tokens as many values as drafts and draws say")
        p = _probs(target, target_ids, target_kept, drafts + seqs, self.vocab, device)
        q = None
        if draft is not None:
            q = _probs(draft, draft_ids, draft_kept, drafts, self.vocab, device)
        _check(lib().rl_drafts_verify(
            self.h, p, q, _index(drafted, torch.int32, drafts, device), _index(starts, torch.int32, seqs + 1, device),
            _index(uniforms, torch.float32, drafts, device), _index(draws, torch.float32, seqs, device), drafts, seqs,
            _index(accepted, torch.int32, seqs, device), _index(tokens, torch.int32, drafts + seqs, device),
            _stream(device, stream)))
