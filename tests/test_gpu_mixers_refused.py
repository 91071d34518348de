"""A refusal leaves nothing behind: what fails in a create call is reported there,
and not by the next launch, this library's or torch's."""
import pytest
import torch

import mixer_fixtures as F
import rl_mixers as M
import rl_sampler as R

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("what", ["memory", "device"])
def test_what_a_create_call_reports_is_reported_once(device, what):
    rotary = M.DeviceRotary(16)
    x, at = torch.ones(3, 2, 16, device=device), torch.arange(3, device=device)
    want = torch.empty_like(x)
    rotary.apply(x, at, want)
    torch.cuda.synchronize()
    for first in ("library", "torch"):
        with pytest.raises(R.SamplerError) as e:
            if what == "memory":
                M.DeviceCache(2 ** 16, 2 ** 16, 64, 256, "bf16")  # 2^47 bytes of keys
            else:
                M.DeviceRotary(16, device=99)
        assert e.value.code == R.RL_ERR_DEVICE
        if first == "torch":
            assert float((x + 1).sum()) == 192.0
        got = torch.empty_like(x)
        rotary.apply(x, at, got)
        torch.cuda.synchronize()
        assert torch.equal(got, want) and F.as64(got).shape == (3, 2, 16)
