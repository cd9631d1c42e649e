"""Dense attention over a shared prefix against a plain form in 64 bits.

Tolerances, for inputs of standard normal values and scale 1/24:

* a score is 576 products summed in 32 bits, at most 50 roundings deep
  (18 products of 32, and the sum inside one), so off by 50 x 2^-24 x
  sum|q k| x scale < 2^-14 (sum|q k| is about 370, below 480);
* a weight exp(score - max) has the errors of two scores, below 2^-13, and the
  sums of weights add below 2^-13 more (n x 2^-24 over a piece of n <= 2048
  keys): max within 2^-14, sum within 2^-12 of itself;
* the output adds the rounding of each weight to bf16, half a step, 2^-8 of it,
  and its own, 2^-8: within (2^-8 + 2^-12) (sum w|v| / sum w + |out|).
"""
import math

import pytest
import torch

import dsa_amd

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm GPU")
    torch.cuda.init()


def make(B, SQ, H, P, S, block=0, fp8=False, seed=0, spare=0):
    """A batch whose rows [0, P) are the same, with S more of each sequence's
    own, in one of the three cache layouts; ``rows [B, L, 576]`` in 64 bits."""
    g = torch.Generator().manual_seed(seed)
    L = P + S
    if block:
        L = -(-L // block) * block
    kv, kr = torch.randn(B, L, 512, generator=g).bfloat16(), torch.randn(B, L, 64, generator=g).bfloat16()
    kv[:, :P], kr[:, :P] = kv[:1, :P].clone(), kr[:1, :P].clone()
    q, qr = torch.randn(B, SQ, H, 512, generator=g).bfloat16(), torch.randn(B, SQ, H, 64, generator=g).bfloat16()
    table = None
    if fp8:
        packed = dsa_amd.quantize_kv_fp8(kv, kr)
        codes = packed[..., :512].contiguous().view(torch.float8_e4m3fn).double()
        scale = packed[..., 512:528].contiguous().view(torch.float32).double()
        rows = torch.cat([(codes.unflatten(-1, (4, 128)) * scale[..., None]).flatten(-2), kr.double()], -1)
        store = [packed]
    else:
        rows = torch.cat([kv, kr], -1).double()
        store = [kv, kr]
    if block:
        M = L // block
        table = (torch.randperm(B * M + spare, generator=g)[:B * M]).int().reshape(B, M)
        pools = []
        for t in store:
            pool = torch.zeros(B * M + spare, block, t.shape[-1], dtype=t.dtype)
            pool[table.long().flatten()] = t.reshape(B * M, block, -1)
            pools.append(pool)
        store = pools
    store = [t.unsqueeze(2).contiguous().cuda() for t in store] + ([None] if fp8 else [])
    return dict(q=q.cuda(), q_rope=qr.cuda(), kv=store[0], k_rope=store[1], rows=rows.cuda(),
                table=None if table is None else table.cuda(), P=P, L=L)


def call(s, lengths, prefix=None, **kw):
    return dsa_amd.forward_shared(s["q"], s["kv"], s["q_rope"], s["k_rope"], lengths, s["P"] if prefix is None else prefix,
                                  block_table=s["table"], **kw)


def exact(s, lengths, scale=1 / 24, live=None):
    """out, max, sum and sum w|v| / sum w in 64 bits; ``live [B, L]``: rows behind a usable block entry."""
    B, SQ, H, _ = s["q"].shape
    out = torch.zeros(B, SQ, H, 512, dtype=torch.float64, device="cuda")
    size, top = torch.zeros_like(out), torch.full((B, 1, SQ, H), -math.inf, dtype=torch.float64, device="cuda")
    total = torch.zeros_like(top)
    q = torch.cat([s["q"], s["q_rope"]], -1).double()
    for b in range(B):
        for t in range(SQ):
            n = min(max(int(lengths[b, t]), 0), s["L"])
            rows = s["rows"][b, :n]
            if live is not None:
                rows = rows[live[b, :n]]
            if rows.shape[0] == 0:
                continue
            score = q[b, t] @ rows.t().contiguous() * scale
            m = score.amax(-1)
            w = torch.exp(score - m[:, None])
            v = rows[:, :512].contiguous()
            total[b, 0, t], top[b, 0, t] = w.sum(-1), m
            out[b, t] = w @ v / w.sum(-1)[:, None]
            size[b, t] = w @ v.abs() / w.sum(-1)[:, None]
    return out, top, total, size


def check(got, s, lengths, scale=1 / 24, live=None, sharp=1.0):
    out, top, total = got
    ref, rtop, rtotal, size = exact(s, lengths, scale, live)
    assert out.dtype == torch.bfloat16 and out.shape == ref.shape and top.shape == rtop.shape
    empty = rtotal == 0
    assert torch.equal(top == -math.inf, empty) and torch.equal(total == 0, empty)
    assert not out[empty.squeeze(1)].any()
    wide = sharp * scale * 24  # scores, and their errors, grow with the scale and the queries
    bound = (2.0 ** -8 + 2.0 ** -12 * wide) * (size + ref.abs()) + 1e-30
    assert ((out.double() - ref).abs() <= bound).all(), ((out.double() - ref).abs() / bound).max()
    live_rows = ~empty
    assert ((top.double() - rtop).abs()[live_rows] <= 2.0 ** -14 * wide).all()
    assert ((total.double() / rtotal - 1).abs()[live_rows] <= 2.0 ** -12 * wide).all()


def causal(B, SQ, ends):
    ends = torch.tensor(ends) if not torch.is_tensor(ends) else ends
    return (ends.reshape(-1, 1).expand(B, 1) - (SQ - 1 - torch.arange(SQ))).int().cuda().contiguous()


SHAPES = [
    # B, SQ, H, P, S
    (1, 1, 16, 0, 1), (1, 1, 16, 1, 0), (2, 1, 16, 1, 1), (3, 1, 16, 33, 31), (5, 1, 16, 500, 70), (1, 1, 128, 0, 300),
    (4, 1, 16, 64, 64), (7, 1, 32, 100, 45), (3, 2, 48, 129, 64), (2, 3, 64, 95, 200), (4, 1, 96, 31, 40),
    (2, 4, 128, 257, 130), (1, 7, 16, 0, 90), (3, 33, 16, 40, 33), (2, 50, 64, 70, 50), (1, 1, 16, 0, 5000),
    (64, 1, 16, 300, 20), (2, 1, 16, 4000, 3), (9, 1, 80, 50, 200)]


@pytest.mark.parametrize("layout", ["rows", "paged16", "paged48", "paged7", "fp8", "fp8_paged64", "fp8_paged5"])
@pytest.mark.parametrize("B, SQ, H, P, S", SHAPES)
def test_against_64_bits(B, SQ, H, P, S, layout):
    block = {"paged16": 16, "paged48": 48, "paged7": 7, "fp8_paged64": 64, "fp8_paged5": 5}.get(layout, 0)
    s = make(B, SQ, H, P, S, block, layout.startswith("fp8"), seed=B + P, spare=3)
    g = torch.Generator().manual_seed(S)
    ends = P + S - torch.randint(0, max(1, S - SQ + 1), (B,), generator=g)
    lengths = causal(B, SQ, ends)
    check(call(s, lengths), s, lengths)


@pytest.mark.parametrize("B, SQ, H, P, S", [(5, 2, 16, 100, 60), (4, 1, 16, 256, 64), (3, 3, 128, 70, 50), (6, 1, 64, 40, 40)])
@pytest.mark.parametrize("block", [0, 16])
def test_any_lengths(B, SQ, H, P, S, block):
    """Lengths below the prefix, at its end, none, negative and past the cache, in no order."""
    s = make(B, SQ, H, P, S, block, seed=7)
    picks = [0, 1, P - 1, P, P + 1, -5, s["L"], s["L"] + 1000, 31, 32, 33, P // 2, (1 << 31) - 1, -(1 << 31)]
    for k in range(4):
        g = torch.Generator().manual_seed(k)
        lengths = torch.tensor(picks)[torch.randint(0, len(picks), (B, SQ), generator=g)].int().cuda()
        check(call(s, lengths), s, lengths)
    lengths = torch.zeros(B, SQ, dtype=torch.int32, device="cuda")
    check(call(s, lengths), s, lengths)


@pytest.mark.parametrize("B, SQ, H", [(2100, 1, 16), (700, 2, 64), (530, 1, 48)])
def test_many_sequences(B, SQ, H):
    """More blocks of rows than a workgroup has threads, some of them without keys."""
    s = make(B, SQ, H, 45, 30, seed=B)
    g = torch.Generator().manual_seed(1)
    lengths = torch.randint(-20, 80, (B, SQ), generator=g).int().cuda()
    lengths[100:300] = 0
    check(call(s, lengths), s, lengths)


@pytest.mark.parametrize("fp8", [False, True])
def test_prefix_splits_change_nothing(fp8):
    """The same rows with any part of them called shared."""
    s = make(6, 1, 16, 150, 50, 16, fp8, seed=3)
    lengths = causal(6, 1, torch.tensor([200, 151, 150, 149, 180, 163]))
    for prefix in (0, 1, 16, 31, 100, 149, 150):
        check(call(s, lengths, prefix), s, lengths)


@pytest.mark.parametrize("B, SQ, H", [(4, 1, 16), (3, 4, 16), (2, 2, 64), (2, 1, 128)])
@pytest.mark.parametrize("block", [0, 16])
@pytest.mark.parametrize("poison", [float("nan"), float("inf")])
def test_unseen_rows_may_hold_anything(B, SQ, H, block, poison):
    """NaN and infinities in rows that a query does not see -- behind the
    sequence, or another query's -- leave it as it is."""
    P, S = 70, 45
    s = make(B, SQ, H, P, S, block, seed=11)
    ends = torch.tensor([P + S, P + 3, P, 20][:B])
    lengths = causal(B, SQ, ends)
    want = [t.clone() for t in call(s, lengths)]
    most = lengths.max(1).values.tolist()
    for b in range(B):
        if s["table"] is None:
            rows = s["kv"].view(B, s["L"], 512)[b], s["k_rope"].view(B, s["L"], 64)[b]
            at = torch.arange(s["L"], device="cuda")
        else:
            rows = s["kv"].view(-1, 512), s["k_rope"].view(-1, 64)
            at = (s["table"][b].long()[:, None] * block + torch.arange(block, device="cuda")).flatten()
        hidden = at[max(P, most[b]):]
        rows[0][hidden], rows[1][hidden] = poison, poison
    for a, w in zip(call(s, lengths), want):
        assert torch.equal(a, w)
    if SQ > 1:  # the last query's own newest row: the earlier queries do not see it
        b = 0
        row = lengths[b, -1].item() - 1
        if s["table"] is None:
            s["kv"][b, row], s["k_rope"][b, row] = poison, poison
        else:
            page = s["table"][b, row // block].item()
            s["kv"][page, row % block], s["k_rope"][page, row % block] = poison, poison
        for a, w in zip(call(s, lengths), want):
            a, w = (t.reshape(B, SQ, H, -1) if t.dim() == 4 and t.shape[1] == SQ else t.transpose(1, 2).reshape(B, SQ, H, -1)
                    for t in (a, w))
            assert torch.equal(a[0, :-1], w[0, :-1]) and torch.equal(a[1:], w[1:])


@pytest.mark.parametrize("H", [16, 64, 128])
@pytest.mark.parametrize("block", [16, 64, 3])
@pytest.mark.parametrize("fp8", [False, True])
def test_bad_block_entries_are_masked(fp8, block, H):
    """Entries outside the pool, in the prefix and behind it, hide their rows."""
    s = make(4, 2, H, 96, 64, block, fp8, seed=5, spare=2)
    n, prefix = s["kv"].shape[0], torch.arange(s["L"], device="cuda") < 96
    live = torch.ones(4, s["L"], dtype=torch.bool, device="cuda")
    for b, key, value in [(0, 16, -1), (0, 64, n), (1, 96, (1 << 31) - 1), (2, 112, -(1 << 31)), (3, 144, n + 5)]:
        entry = key // block
        s["table"][b, entry] = value
        rows = torch.arange(s["L"], device="cuda") // block == entry
        live[b, rows & ~prefix] = False
        if b == 0:
            live[:, rows & prefix] = False
    lengths = causal(4, 2, torch.tensor([160, 160, 130, 98]))
    check(call(s, lengths), s, lengths, live=live)
    s["table"].fill_(-1)
    live[:] = False
    check(call(s, lengths), s, lengths, live=live)


def test_growing_scores():
    """Scores that rise far along the keys (2^100 from the first tile's weights
    to the last one's), and ones that fall: the maximum found on the way."""
    for B, H, P, S in [(3, 16, 200, 100), (2, 128, 150, 90)]:
        s = make(B, 1, H, P, S, seed=2)
        ramp = torch.linspace(-1, 1, P + S, device="cuda")
        for sign in (1, -1):
            q = torch.ones_like(s["q"][..., :1]) * 40
            s["q"][..., :1] = q
            s["kv"][..., 0, 0] = (sign * ramp * 30).bfloat16()
            s["rows"][..., 0] = s["kv"][..., 0, 0].double()
            lengths = causal(B, 1, torch.full((B,), P + S))
            # a score now holds a product up to 1200 beside the 480: 3.5 times the errors
            check(call(s, lengths), s, lengths, sharp=3.5)


def test_scale():
    s = make(3, 1, 16, 40, 20, seed=9)
    lengths = causal(3, 1, torch.tensor([60, 50, 41]))
    for scale in (192 ** -0.5, 0.01, 1):
        check(call(s, lengths, scale=scale), s, lengths, scale=scale)


def test_agrees_with_the_sparse_kernels():
    """The same rows as forward() with every row selected."""
    s = make(2, 3, 128, 300, 212, 64, seed=21)
    lengths = causal(2, 3, torch.tensor([512, 480]))
    ids = torch.arange(s["L"], dtype=torch.int32, device="cuda").expand(2, 3, 1, s["L"]).clone()
    ids[ids >= lengths[:, :, None, None]] = -1
    for fp8 in (False, True):
        if fp8:
            s["kv"], s["k_rope"] = dsa_amd.quantize_kv_fp8(s["kv"], s["k_rope"]), None
        a = call(s, lengths)
        b = dsa_amd.forward(s["q"], s["kv"], s["q_rope"], s["k_rope"], ids, block_table=s["table"])
        # two results of the same bf16 weights' order of rounding: a step each
        assert (a[0].float() - b[0].float()).abs().max() <= 2.0 ** -7 * b[0].float().abs().max()
        assert (a[1] - b[1]).abs().max() <= 2.0 ** -13 and ((a[2] / b[2]) - 1).abs().max() <= 2.0 ** -11


def test_far_offsets():
    """Rows past 4 GiB of a contiguous cache, and of a pool."""
    B, L = 2200, 2048
    kv = torch.zeros(B, L, 1, 512, device="cuda", dtype=torch.bfloat16)
    kr = torch.zeros(B, L, 1, 64, device="cuda", dtype=torch.bfloat16)
    g = torch.Generator(device="cuda").manual_seed(0)
    n = 45
    kv[:, :n] = torch.randn(B, n, 1, 512, device="cuda", generator=g).bfloat16()
    kr[:, :n] = torch.randn(B, n, 1, 64, device="cuda", generator=g).bfloat16()
    q = torch.randn(B, 1, 16, 512, device="cuda", generator=g).bfloat16()
    qr = torch.randn(B, 1, 16, 64, device="cuda", generator=g).bfloat16()
    lengths = torch.full((B, 1), n, dtype=torch.int32, device="cuda")
    pick = [0, 1, 1030, 2100, B - 1]
    s = dict(q=q[pick].contiguous(), q_rope=qr[pick].contiguous(), L=n,
             rows=torch.cat([kv[pick, :n, 0], kr[pick, :n, 0]], -1).double())
    got = dsa_amd.forward_shared(q, kv, qr, kr, lengths)
    check([got[0][pick], got[1][pick], got[2][pick]], s, lengths[pick])
    # as a pool of 64-row blocks, the last sequences' blocks at its end
    pool, rpool = kv.view(B * L // 64, 64, 1, 512), kr.view(B * L // 64, 64, 1, 64)
    table = (torch.arange(B, device="cuda").int() * (L // 64))[:, None].contiguous()
    got = dsa_amd.forward_shared(q, pool, qr, rpool, lengths, block_table=table)
    check([got[0][pick], got[1][pick], got[2][pick]], s, lengths[pick])


def test_long_context():
    """One query over 200,000 rows, cut over every workgroup."""
    L = 200001
    g = torch.Generator(device="cuda").manual_seed(4)
    kv = torch.randn(1, L, 1, 512, device="cuda", generator=g).bfloat16()
    kr = torch.randn(1, L, 1, 64, device="cuda", generator=g).bfloat16()
    q, qr = (torch.randn(1, 1, 16, d, device="cuda", generator=g).bfloat16() for d in (512, 64))
    s = dict(q=q, q_rope=qr, L=L, rows=torch.cat([kv, kr], -1)[:, :, 0].double())
    for n in (L, L - 1, 100000):
        lengths = torch.full((1, 1), n, dtype=torch.int32, device="cuda")
        check(dsa_amd.forward_shared(q, kv, qr, kr, lengths), s, lengths)


def test_repeats_are_the_same_bits():
    s = make(8, 1, 16, 700, 100, 16, seed=13)
    lengths = causal(8, 1, torch.arange(793, 801))
    first = call(s, lengths)
    for _ in range(3):
        for a, b in zip(first, call(s, lengths)):
            assert torch.equal(a, b)


def test_streams_and_graphs():
    """Two graphs and eager calls on two streams, replayed in turn: nothing is shared between them."""
    a, b = make(4, 1, 16, 300, 40, 16, seed=1), make(2, 2, 128, 90, 30, seed=2)
    la, lb = causal(4, 1, torch.tensor([340, 320, 310, 301])), causal(2, 2, torch.tensor([120, 100]))
    call(a, la), call(b, lb)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs = []
    for s, lengths in ((a, la), (b, lb)):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call(s, lengths)
        graphs.append((graph, out))
    for k in range(4):
        la.copy_(torch.randint(0, 341, (4, 1)))
        a["q"].copy_(torch.randn(a["q"].shape))
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            other = call(b, lb)
        graphs[0][0].replay()
        graphs[1][0].replay()
        torch.cuda.synchronize()
        for s, lengths, out in ((a, la, graphs[0][1]), (b, lb, graphs[1][1]), (b, lb, other)):
            for x, y in zip(out, call(s, lengths)):
                assert torch.equal(x, y)
            check(out, s, lengths)


def test_refusals():
    s = make(2, 1, 16, 16, 16, seed=0)
    lengths = causal(2, 1, torch.tensor([32, 20]))
    good = dict(q=s["q"], kv=s["kv"], q_rope=s["q_rope"], k_rope=s["k_rope"], lengths=lengths, prefix=16)
    dsa_amd.forward_shared(**good)
    rows = dsa_amd.quantize_kv_fp8(s["kv"], s["k_rope"])
    table = torch.zeros(2, 2, dtype=torch.int32, device="cuda")
    q24 = torch.zeros(2, 1, 24, 512, device="cuda", dtype=torch.bfloat16)
    bad = [dict(q=s["q"].float()), dict(q=s["q"][0]), dict(q=q24, q_rope=q24[..., :64].contiguous()), dict(kv=s["kv"].half()),
           dict(kv=s["kv"][:1]), dict(kv=s["kv"].cpu()), dict(kv=rows), dict(k_rope=None), dict(k_rope=s["k_rope"][:, :-1]),
           dict(q_rope=s["q_rope"][..., :32]), dict(lengths=lengths.long()), dict(lengths=lengths[:1]),
           dict(lengths=lengths.cpu()), dict(prefix=-1), dict(prefix=33), dict(prefix=1.0), dict(scale=0.0),
           dict(scale=float("inf")), dict(block_table=table.long()), dict(block_table=table[:1]), dict(block_table=table[0]),
           dict(block_table=table.cpu()), dict(q=s["q"].transpose(1, 2).expand(2, 16, 16, 512)),
           dict(kv=s["kv"].transpose(0, 1)), dict(q=s["q"][:0], q_rope=s["q_rope"][:0], lengths=lengths[:0])]
    for kw in bad:
        with pytest.raises(ValueError):
            dsa_amd.forward_shared(**{**good, **kw})
    with pytest.raises(TypeError):
        dsa_amd.forward_shared(**good, scale="1")


# ------------------------------------------------------------ the operators together

@pytest.mark.parametrize("fp8", [False, True])
def test_serving_steps(fp8):
    """A shared prompt is written once; three requests behind it get a prompt of
    their own and then decode, each step by the four operators; every step's
    attention equals that over rows kept on the side in plain tensors."""
    B, H, block, width, P = 3, 16, 16, 24, 64
    g = torch.Generator().manual_seed(0)
    blocks = B * width
    freq = dsa_amd.rotary_frequencies(64, scaling="yarn", factor=4.0).cuda()
    if fp8:
        pools = (torch.zeros(blocks, block, 1, 656, dtype=torch.uint8, device="cuda"), None)
    else:
        pools = (torch.zeros(blocks, block, 1, 512, dtype=torch.bfloat16, device="cuda"),
                 torch.zeros(blocks, block, 1, 64, dtype=torch.bfloat16, device="cuda"))
    free = torch.randperm(blocks, generator=g).int().cuda()
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    kept = [[] for _ in range(B)]

    def rows(n):
        return torch.randn(n, 512, generator=g).bfloat16().cuda(), torch.randn(n, 576, generator=g).bfloat16().cuda()[:, 512:]

    def turned(x, positions):
        """The rotation in plain torch, rounded once."""
        angle = positions.double()[:, None] * freq
        z = torch.view_as_complex(x.double().unflatten(-1, (-1, 2)).contiguous())
        turn = torch.polar(torch.ones_like(angle), angle)
        return torch.view_as_real(z * (turn if x.dim() == 2 else turn[:, None])).flatten(-2).bfloat16()

    def remember(b, kv, rope):
        r = dsa_amd.quantize_kv_fp8(kv, rope) if fp8 else None
        if fp8:
            codes = r[:, :512].contiguous().view(torch.float8_e4m3fn).double().unflatten(-1, (4, 128))
            kv = (codes * r[:, 512:528].contiguous().view(torch.float32).double()[..., None]).flatten(-2)
        kept[b].append(torch.cat([kv.double(), rope.double()], -1))

    # the shared prompt, in sequence 0's row, then that row's blocks in every row
    table = torch.full((B, width), -1, dtype=torch.int32, device="cuda")
    kv, rope = rows(P)
    first = table[:1].clone()
    slots, positions, _, totals, used = dsa_amd.extend_block_table(first, i32(0), i32(P), free, block, P)
    dsa_amd.write_kv_rows(kv, rope, slots, *pools, positions=positions, frequencies=freq)
    table[:, :P // block] = first[:, :P // block]
    free = free[int(used):].contiguous()
    for b in range(B):
        remember(b, kv, turned(rope, positions))
    lengths = totals.expand(B).contiguous()
    for step in range(6):
        new = i32(19, 0, 33) if step == 0 else i32(1, 1, 1)
        most = int(new.sum())
        slots, positions, starts, lengths, used = dsa_amd.extend_block_table(table, lengths, new, free, block, most)
        free = free[int(used):].contiguous()
        kv, rope = rows(most)
        dsa_amd.write_kv_rows(kv, rope, slots, *pools, positions=positions, frequencies=freq)
        at = starts.tolist()
        for b in range(B):
            p = positions[at[b]:at[b + 1]]
            if p.numel():
                remember(b, kv[at[b]:at[b + 1]], turned(rope[at[b]:at[b + 1]], p))
        SQ = 33 if step == 0 else 1
        q = torch.randn(B, SQ, H, 512, generator=g).bfloat16().cuda()
        raw = torch.randn(B, SQ, H, 192, generator=g).bfloat16().cuda()
        # the last queries of each sequence; padding in front of the shorter ones sees nothing
        spot = lengths[:, None] - SQ + torch.arange(SQ, device="cuda").int()
        seen = torch.where(spot >= lengths[:, None] - new[:, None], spot + 1, 0).int()
        spot = spot.clamp_min(0).contiguous()
        q_rope = dsa_amd.rotary(raw[..., 128:], spot, freq)
        want = turned(raw[..., 128:].reshape(B * SQ, H, 64), spot.flatten()).view(B, SQ, H, 64)
        # the two round to bf16 from values 2^-20 apart
        assert (q_rope.float() - want.float()).abs().max() <= 2.0 ** -7 * want.float().abs().max()
        got = dsa_amd.forward_shared(q, pools[0], q_rope, pools[1], seen, P, block_table=table)
        L = int(lengths.max())
        side = torch.zeros(B, L, 576, dtype=torch.float64, device="cuda")
        for b in range(B):
            r = torch.cat(kept[b])
            side[b, :r.shape[0]] = r
        s = dict(q=q, q_rope=q_rope, L=L, rows=side)
        # rope values of the side rows may be a rounding step (2^-8 of them) from the cache's, in 64 of 576
        # products: scores off by 2^-8 x 64 x 0.64 / 24 = 2^-7.2 at worst, were every value to differ
        ref = exact(s, seen)
        assert ((got[0].double() - ref[0]).abs() <= 2.0 ** -6 * (ref[3] + ref[0].abs())).all()
        assert torch.equal(got[2] == 0, seen[:, None, :, None].expand_as(got[2]) == 0)
