"""The handles of the token mixers hold no more memory than include/rl_mixers.h says."""
import gc

import pytest
import torch

import rl_mixers as M

pytestmark = pytest.mark.gpu


def held(make):
    """Device bytes that a handle takes."""
    gc.collect()
    torch.cuda.synchronize()
    before = torch.cuda.mem_get_info()[0]
    h = make()
    after = torch.cuda.mem_get_info()[0]
    h.close()
    return before - after


DELTA = [
    # max_rows, max_seqs, key heads, value heads, key dim, value dim
    (8192, 64, 16, 32, 128, 128),
    (2048, 4, 8, 8, 256, 64),
    (640, 1000, 4, 16, 48, 96),
]


@pytest.mark.parametrize("sizes", DELTA)
def test_delta_workspace(device, sizes):
    rows, seqs, kh, vh, dk, _ = sizes
    chunks = rows // 64 + min(seqs, rows // 16 + 1)
    wide = 64 if dk <= 64 else 128 if dk <= 128 else 256
    want = chunks * (vh * 41 * 1024 + kh * 768 * wide)
    held(lambda: M.DeviceDelta(*sizes))  # the first call may load code
    got = held(lambda: M.DeviceDelta(*sizes))
    # Six allocations, each in pieces of up to 2 MiB. (Small ones may take none: they share pieces with others.)
    assert got <= want + 6 * 2 ** 21, (got, want)


ATTEND = [
    # max_rows, q heads, kv heads, dim, max_len
    (8192, 32, 8, 128, 131072),
    (64, 32, 8, 128, 8192),
    (1, 8, 1, 80, 10 ** 9),
    (16384, 64, 4, 256, 2 ** 20),
]


@pytest.mark.parametrize("sizes", ATTEND)
def test_attention_workspace(device, sizes):
    rows, heads, _, dim, length = sizes
    parts = min(length // 1536 + 1, 256)
    wide = 64 if dim <= 64 else 128 if dim <= 128 else 256
    want = rows * heads * 8 + max(min(rows * heads * parts, 2 ** 20), 24576) * (4 * wide + 8)
    held(lambda: M.DeviceAttention(*sizes))
    got = held(lambda: M.DeviceAttention(*sizes))
    assert got <= want + 4 * 2 ** 21, (got, want)
