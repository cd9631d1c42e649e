"""Calls of the paged cache's operators that one launch does not hold: more than
2^32 threads.  Each is many copies of a small call, whose results it has to equal."""
import pytest
import torch

import dsa_amd

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm GPU")
    torch.cuda.init()


@pytest.mark.parametrize("groups", [1, 3])
def test_rotary_of_more_workgroups_than_a_launch(groups):
    """2^24 and some tokens of 256 units (nothing aligned: a pair each), a workgroup a token: 17 GB, in place."""
    period, tokens = 4096, (1 << 24) + 5
    freq = dsa_amd.rotary_frequencies(64).cuda()
    base = torch.empty(period * 512 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(period, 8, 64)
    base.copy_(torch.randn(period, 8, 64, generator=torch.Generator().manual_seed(0)).bfloat16())
    want = dsa_amd.rotary(base, torch.arange(period, device="cuda"), freq)
    x = torch.empty(tokens * 512 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(tokens, 8, 64)
    x[:1 << 24].view(-1, period, 8, 64).copy_(base)
    x[1 << 24:] = base[:5]
    positions = (torch.arange(tokens, device="cuda") % period).int()
    print("rotary", tokens, groups, flush=True)
    dsa_amd.rotary(x.view(groups, -1, 8, 64), positions.view(groups, -1), freq, out=x.view(groups, -1, 8, 64))
    for block in x[:1 << 24].view(-1, 256 * period, 8, 64):
        assert torch.equal(block.view(256, period, 8, 64), want.expand(256, -1, -1, -1))
    assert torch.equal(x[1 << 24:], want[:5])
