"""What the handles of the token mixers hold is what include/rl_mixers.h says."""
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
    # Six allocations, each in pieces of up to 2 MiB.
    assert want <= got <= want + 6 * 2 ** 21, (got, want)
