"""Calls of the paged cache's operators that one launch does not hold: more than
2^32 threads.  Each is many copies of a small call, whose results it has to equal."""
import pytest
import torch

import dsa_amd
from test_gpu_shared_pieces import run

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


def test_attention_of_more_blocks_than_a_launch():
    """2^21 sequences of one key and 16 heads, some of them padding: 73 GB of queries
    and outputs, each output its sequence's row."""
    B = (1 << 21) + 9
    g = torch.Generator(device="cuda").manual_seed(0)
    kv = torch.randn(B, 1, 1, 512, generator=g, device="cuda", dtype=torch.bfloat16)
    q = torch.empty(B, 1, 16, 512, device="cuda", dtype=torch.bfloat16)
    q.copy_(torch.randn(16, 512, generator=g, device="cuda"))
    s = dict(q=q, q_rope=torch.zeros(B, 1, 16, 64, device="cuda", dtype=torch.bfloat16), kv=kv, table=None, L=1,
             k_rope=torch.zeros(B, 1, 1, 64, device="cuda", dtype=torch.bfloat16))
    lengths = torch.ones(B, 1, dtype=torch.int32, device="cuda")
    empty = torch.tensor([0, 7, 1 << 20, (1 << 21) - 1, 1 << 21, B - 1], device="cuda")
    lengths[empty] = 0
    kv[empty] = 0
    print("attention", B, flush=True)
    out, top, total = run(s, lengths, 256, 0)
    for a, b in zip(out.split(1 << 17), kv.split(1 << 17)):
        assert torch.equal(a, b.expand_as(a))
    assert torch.equal(total, lengths.view(B, 1, 1, 1).float().expand_as(total))
    assert (top[empty] == -float("inf")).all() and int(top.isinf().sum()) == 16 * empty.numel()
