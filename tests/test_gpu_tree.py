"""Drafted trees: ancestors against a walk on the host, and their attention against a
plain form in 64 bits, with the tolerances of dense attention (tests/test_gpu_shared.py)."""
import math
import random

import pytest
import torch

import dsa_amd
from test_gpu_shared import make

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm GPU")
    torch.cuda.init()


def i32(v):
    return torch.tensor(v, dtype=torch.int32).cuda()


# ------------------------------------------------------------ draft_tree

def walk(parents, length):
    bits, places = [], []
    for t, parent in enumerate(parents):
        if parent < -1 or parent >= t or (parent >= 0 and bits[parent] == 0):
            bits.append(0)
            places.append(0)
        else:
            bits.append(1 << t | (bits[parent] if parent >= 0 else 0))
            places.append(min(max(length, 0) + bin(bits[t]).count("1") - 1, 2 ** 31 - 1))
    words = -(-len(parents) // 32)
    signed = lambda v: v - (1 << 32) if v >> 31 else v  # noqa: E731
    return [[signed(m >> 32 * w & 0xFFFFFFFF) for w in range(words)] for m in bits], places


@pytest.mark.parametrize("B, SQ", [(1, 1), (3, 7), (64, 8), (2, 31), (2, 32), (5, 33), (1, 64), (3, 100), (2, 257), (1, 1000),
                                   (2, 2048), (300, 5)])
def test_ancestors(B, SQ):
    rng = random.Random(B + SQ)
    kinds = [lambda t: rng.randint(-1, t - 1) if t else -1,      # any tree
             lambda t: t - 1,                                    # a line
             lambda t: -1,                                       # all on the sequence
             lambda t: rng.choice([rng.randint(-1, max(-1, t - 1)), -2, t, t + 1, 2 ** 31 - 1, -2 ** 31])]  # padding among them
    parents = [[kinds[b % 4](t) for t in range(SQ)] for b in range(B)]
    lengths = [rng.choice([0, 1, 77, -3, 2 ** 31 - 1, 30000]) for _ in range(B)]
    tree, positions = dsa_amd.draft_tree(i32(parents), i32(lengths))
    want = [walk(p, n) for p, n in zip(parents, lengths)]
    assert tree.dtype == positions.dtype == torch.int32
    assert tree.tolist() == [w[0] for w in want] and positions.tolist() == [w[1] for w in want]


# ------------------------------------------------------------ forward_tree

def tree_of(bits):
    """Words of a truth table [B, SQ, n]."""
    words = -(-bits.shape[-1] // 32)
    wide = torch.nn.functional.pad(bits.long(), (0, words * 32 - bits.shape[-1])).unflatten(-1, (words, 32))
    value = (wide << torch.arange(32)).sum(-1)
    return torch.where(value >= 1 << 31, value - (1 << 32), value).int().cuda()


def random_bits(B, SQ, n, seed):
    return torch.rand(B, SQ, n, generator=torch.Generator().manual_seed(seed)) < 0.5


def seen_rows(s, lengths, bits):
    """[B, SQ, L]: what each query sees."""
    at = torch.arange(s["L"]) - lengths.cpu().long().clamp(0, s["L"])[:, None]
    drafted = bits.gather(2, at.clamp(0, bits.shape[2] - 1)[:, None].expand(-1, bits.shape[1], -1))
    return ((at < 0)[:, None] | (((at >= 0) & (at < bits.shape[2]))[:, None] & drafted)).cuda()


def check(got, s, seen, scale=1 / 24):
    out, top, total = got
    B, SQ, H, _ = s["q"].shape
    q = torch.cat([s["q"], s["q_rope"]], -1).double()
    for b in range(B):
        rows = s["rows"][b]
        score = (q[b].view(SQ * H, 576) @ rows.t().contiguous()).view(SQ, H, -1) * scale
        score.masked_fill_(~seen[b][:, None], -math.inf)
        m = score.amax(-1)
        empty = ~seen[b].any(-1)
        w = torch.exp(score - torch.where(m > -math.inf, m, 0.0)[..., None])
        norm = w.sum(-1)
        safe = torch.where(norm > 0, norm, 1.0)[..., None]
        v = rows[:, :512].contiguous()
        ref = (w.view(SQ * H, -1) @ v).view(SQ, H, 512) / safe
        size = (w.view(SQ * H, -1) @ v.abs()).view(SQ, H, 512) / safe
        assert not out[b][empty].any() and (top[b, 0][empty] == -math.inf).all() and not total[b, 0][empty].any()
        bound = (2.0 ** -8 + 2.0 ** -12) * (size + ref.abs()) + 1e-30
        assert ((out[b].double() - ref).abs() <= bound).all()
        live = ~empty
        assert ((top[b, 0].double() - m).abs()[live] <= 2.0 ** -14).all()
        assert ((total[b, 0].double() / safe[..., 0] - 1).abs()[live] <= 2.0 ** -12).all()


def call(s, lengths, tree, prefix=None, **kw):
    return dsa_amd.forward_tree(s["q"], s["kv"], s["q_rope"], s["k_rope"], lengths, tree, s["P"] if prefix is None else prefix,
                                block_table=s["table"], **kw)


SHAPES = [
    # B, SQ, H, P, S (context and drafts), most drafted rows
    (1, 1, 16, 0, 1, 1), (1, 1, 16, 0, 40, 1), (2, 3, 16, 5, 30, 3), (3, 7, 16, 33, 60, 7), (1, 5, 128, 0, 200, 5),
    (4, 2, 64, 64, 64, 31), (2, 9, 48, 100, 70, 33), (3, 33, 16, 40, 90, 33), (1, 60, 32, 0, 150, 60), (2, 17, 80, 31, 130, 64),
    (1, 70, 16, 10, 120, 70), (2, 8, 128, 257, 130, 100), (1, 4, 16, 0, 5000, 64), (20, 4, 16, 300, 50, 8),
    (1, 3, 16, 4, 2200, 2048)]


@pytest.mark.parametrize("layout", ["rows", "paged16", "paged7", "fp8", "fp8_paged64", "fp8_paged5"])
@pytest.mark.parametrize("B, SQ, H, P, S, n", SHAPES)
def test_against_64_bits(B, SQ, H, P, S, n, layout):
    """Any bits, not only a tree's, behind any length from the prefix on."""
    block = {"paged16": 16, "paged7": 7, "fp8_paged64": 64, "fp8_paged5": 5}.get(layout, 0)
    s = make(B, SQ, H, P, S, block, layout.startswith("fp8"), seed=B + P, spare=3)
    g = torch.Generator().manual_seed(S)
    lengths = (P + torch.randint(0, max(1, S - n + 1), (B,), generator=g)).int().cuda()
    bits = random_bits(B, SQ, n, seed=n)
    check(call(s, lengths, tree_of(bits)), s, seen_rows(s, lengths, bits))


@pytest.mark.parametrize("B, SQ, H, P, S", [(5, 2, 16, 100, 60), (4, 6, 16, 256, 64), (3, 9, 128, 70, 50), (6, 4, 64, 40, 40)])
@pytest.mark.parametrize("block", [0, 16])
def test_any_lengths(B, SQ, H, P, S, block):
    """Lengths of none, negative, inside the prefix, at the cache's end and past it; queries without a bit."""
    s = make(B, SQ, H, P, S, block, seed=7)
    picks = [0, 1, P - 1, P, P + 1, -5, s["L"], s["L"] - 1, s["L"] - 3, s["L"] + 1000, 31, 32, 33, (1 << 31) - 1, -(1 << 31)]
    for k in range(4):
        g = torch.Generator().manual_seed(k)
        lengths = torch.tensor(picks)[torch.randint(0, len(picks), (B,), generator=g)].int().cuda()
        bits = random_bits(B, SQ, 40, seed=k)
        bits[torch.rand(B, SQ, generator=g) < 0.3] = False
        check(call(s, lengths, tree_of(bits)), s, seen_rows(s, lengths, bits))
    lengths = torch.zeros(B, dtype=torch.int32, device="cuda")
    bits = torch.zeros(B, SQ, 7, dtype=torch.bool)
    check(call(s, lengths, tree_of(bits)), s, seen_rows(s, lengths, bits))


def test_a_line_is_causal():
    """A tree that is a line sees what causal lengths give."""
    s = make(3, 20, 16, 40, 60, 16, seed=2)
    lengths = i32([60, 41, 80])
    parents = i32([[t - 1 for t in range(20)]] * 3)
    tree, positions = dsa_amd.draft_tree(parents, lengths)
    causal = (lengths[:, None] + torch.arange(1, 21, device="cuda")).int()
    assert torch.equal(positions + 1, causal)
    got = call(s, lengths, tree)
    want = dsa_amd.forward_shared(s["q"], s["kv"], s["q_rope"], s["k_rope"], causal, 40, block_table=s["table"])
    for a, b in zip(got, want):
        assert torch.allclose(a.float(), b.float(), rtol=2.0 ** -7, atol=2.0 ** -9)


@pytest.mark.parametrize("B, SQ, H", [(2, 4, 16), (2, 3, 64), (2, 5, 128)])
@pytest.mark.parametrize("block", [0, 16, 5])
@pytest.mark.parametrize("poison", [float("nan"), float("inf")])
def test_unseen_rows_may_hold_anything(B, SQ, H, block, poison):
    """Another branch's rows, and rows behind the tree, leave a query as it is; its own do what the formulas say."""
    s = make(B, SQ, H, 20, 75, block, seed=11)
    lengths = i32([40, 61])
    bits = torch.zeros(B, SQ, SQ, dtype=torch.bool)
    for t in range(SQ):
        bits[:, t, t] = True
        if t > 1:
            bits[:, t, t - 2] = True
    want = [t.clone() for t in call(s, lengths, tree_of(bits))]
    for b in range(B):
        n = int(lengths[b])
        if s["table"] is None:
            at = b * s["L"] + torch.arange(s["L"], device="cuda")
        else:
            at = (s["table"][b].long()[:, None] * block + torch.arange(block, device="cuda")).flatten()
        hidden = torch.cat([at[n + 1:n + 2], at[n + SQ:]])  # the second token's row: seen by the odd ones
        s["kv"].view(-1, 512)[hidden], s["k_rope"].view(-1, 64)[hidden] = poison, poison
    got = call(s, lengths, tree_of(bits))
    for a, w in zip(got, want):
        a, w = (a, w) if a.shape[1] == SQ else (a[:, 0], w[:, 0])
        assert torch.equal(a[:, 0], w[:, 0])
        if SQ > 2:
            assert torch.equal(a[:, 2], w[:, 2])
    assert got[0][:, 1].isnan().all()


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("block", [16, 5])
def test_bad_block_entries_are_masked(fp8, block):
    s = make(3, 6, 16, 0, 90, block, fp8, seed=4, spare=2)
    table = s["table"]
    table[0, 1], table[1, 70 // block], table[2, 0] = -1, s["kv"].shape[0], 2 ** 31 - 1
    lengths = i32([50, 66, 0])
    bits = random_bits(3, 6, 24, seed=1)
    seen = seen_rows(s, lengths, bits)
    row = torch.arange(s["L"], device="cuda") // block
    for b, bad in ((0, 1), (1, 70 // block), (2, 0)):
        seen[b, :, row == bad] = False
    s["rows"][~torch.isfinite(s["rows"])] = 0.0
    check(call(s, lengths, tree_of(bits)), s, seen)


def test_far_block_entries():
    """Pool rows beyond 2^31 bytes from its start."""
    blocks, block = 40000, 64
    kv = torch.zeros(blocks, block, 1, 512, dtype=torch.bfloat16, device="cuda")
    kr = torch.zeros(blocks, block, 1, 64, dtype=torch.bfloat16, device="cuda")
    small = make(2, 5, 16, 0, 128, 64, seed=9)
    table = i32([[39999, 3], [39000, 38000]])
    for b in range(2):
        for j in range(2):
            kv[table[b, j]] = small["kv"][small["table"][b, j]]
            kr[table[b, j]] = small["k_rope"][small["table"][b, j]]
    lengths, bits = i32([100, 61]), random_bits(2, 5, 20, seed=3)
    got = dsa_amd.forward_tree(small["q"], kv, small["q_rope"], kr, lengths, tree_of(bits), block_table=table)
    check(got, small, seen_rows(small, lengths, bits))


def test_scale_and_prefix():
    s = make(4, 5, 16, 90, 60, 16, seed=5)
    lengths, bits = i32([100, 120, 95, 130]), random_bits(4, 5, 20, seed=2)
    seen = seen_rows(s, lengths, bits)
    check(call(s, lengths, tree_of(bits), scale=1 / 30), s, seen, 1 / 30)
    for prefix in (0, 1, 16, 31, 89):
        check(call(s, lengths, tree_of(bits), prefix), s, seen)


def test_many_sequences():
    s = make(700, 2, 16, 45, 30, seed=1)
    g = torch.Generator().manual_seed(1)
    lengths = torch.randint(-20, 80, (700,), generator=g).int().cuda()
    lengths[100:300] = 0
    bits = random_bits(700, 2, 9, seed=4)
    bits[100:200] = False
    check(call(s, lengths, tree_of(bits)), s, seen_rows(s, lengths, bits))


def test_streams_and_graphs():
    """Two captured steps, replayed in turn with new trees and lengths, and one on another stream."""
    steps = []
    for k in range(2):
        s = make(3, 9, 16, 40, 80, 16, seed=k)
        parents, lengths = i32([[(t - 1) // 2 if t else -1 for t in range(9)]] * 3), i32([60, 80, 41])
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            tree, positions = dsa_amd.draft_tree(parents, lengths)
            out = call(s, lengths, tree)
        steps.append((s, parents, lengths, graph, tree, positions, out))
    side = torch.cuda.Stream()
    for k in range(4):
        for s, parents, lengths, graph, *_ in steps:
            rng = random.Random(k)
            parents.copy_(i32([[rng.randint(-1, t - 1) if t else -1 for t in range(9)] for _ in range(3)]))
            lengths.copy_(i32([40 + 7 * k, 99, 70 - k]))
        steps[0][3].replay()
        steps[1][3].replay()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = call(steps[0][0], steps[0][2], dsa_amd.draft_tree(steps[0][1], steps[0][2])[0])
        torch.cuda.synchronize()
        for s, parents, lengths, _, tree, positions, out in steps:
            again = dsa_amd.draft_tree(parents, lengths)
            assert torch.equal(tree, again[0]) and torch.equal(positions, again[1])
            for a, b in zip(out, call(s, lengths, tree)):
                assert torch.equal(a, b)
        for a, b in zip(other, steps[0][6]):
            assert torch.equal(a, b)


def test_refusals():
    s = make(2, 3, 16, 16, 16, seed=0)
    lengths, tree = i32([20, 25]), tree_of(random_bits(2, 3, 3, 0))
    good = dict(q=s["q"], kv=s["kv"], q_rope=s["q_rope"], k_rope=s["k_rope"], lengths=lengths, tree=tree, prefix=16)
    dsa_amd.forward_tree(**good)
    bad = [dict(tree=None), dict(tree=tree.long()), dict(tree=tree.cpu()), dict(tree=tree[:1]), dict(tree=tree[:, :2]),
           dict(tree=tree[..., 0]), dict(tree=tree.expand(2, 3, 2)), dict(tree=tree[..., :0]),
           dict(tree=torch.zeros(2, 3, 65, dtype=torch.int32, device="cuda")), dict(lengths=lengths[:, None].expand(2, 3).contiguous()),
           dict(lengths=lengths[:1]), dict(lengths=lengths.long()), dict(lengths=lengths.cpu()), dict(q=s["q"].float()),
           dict(k_rope=None), dict(prefix=33), dict(prefix=True), dict(scale=0.0)]
    for kw in bad:
        with pytest.raises(ValueError):
            dsa_amd.forward_tree(**{**good, **kw})
    parents = i32([[-1, 0, 0], [-1, -1, 1]])
    for args in [(None, lengths), (parents, None), (parents[0], lengths), (parents, lengths[:1]), (parents.long(), lengths),
                 (parents, lengths.long()), (parents.cpu(), lengths), (parents, lengths.cpu()), (parents.t(), i32([1, 2, 3])),
                 (parents[:0], lengths[:0]), (parents[:, :0], lengths), (torch.zeros(1, 2049, dtype=torch.int32).cuda(), lengths[:1])]:
        with pytest.raises(ValueError):
            dsa_amd.draft_tree(*args)
