"""Infinities, NaN and huge scores in rows that queries of forward_shared see,
and in fp8 and odd-block rows that they do not.

The reference is the formula itself in 64 bits, sequence by sequence, products
with infinities included: which elements are NaN and which statistics are
infinite has to agree exactly.  Finite elements keep the tolerance of
test_gpu_shared.py (its derivation covers any subset of keys: a key of weight 0
adds nothing)."""
import math

import pytest
import torch

import dsa_amd

pytestmark = pytest.mark.gpu

INF, NAN = math.inf, math.nan
# layout: block size (0: contiguous), fp8 rows
LAYOUTS = {"rows": (0, False), "paged16": (16, False), "paged7": (7, False), "fp8": (0, True), "fp8_paged16": (16, True),
           "fp8_paged7": (7, True)}


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm GPU")
    torch.cuda.init()


def make(B, SQ, H, L, layout, edit, seed=0):
    """Inputs of L rows a sequence, changed by ``edit(kv, k_rope)`` or
    ``edit(rows)`` (fp8: the packed bytes) before they are laid out."""
    block, fp8 = LAYOUTS[layout]
    g = torch.Generator().manual_seed(seed)
    L = -(-L // block) * block if block else L
    kv, kr = torch.randn(B, L, 512, generator=g).bfloat16(), torch.randn(B, L, 64, generator=g).bfloat16()
    q, qr = torch.randn(B, SQ, H, 512, generator=g).bfloat16(), torch.randn(B, SQ, H, 64, generator=g).bfloat16()
    store = [dsa_amd.quantize_kv_fp8(kv, kr)] if fp8 else [kv, kr]
    edit(*store)
    if fp8:
        codes = store[0][..., :512].contiguous().view(torch.float8_e4m3fn).double()
        scale = store[0][..., 512:528].contiguous().view(torch.float32).double()
        rope = store[0][..., 528:].contiguous().view(torch.bfloat16).double()
        rows = torch.cat([(codes.unflatten(-1, (4, 128)) * scale[..., None]).flatten(-2), rope], -1)
    else:
        rows = torch.cat([kv.double(), kr.double()], -1)
    table = None
    if block:
        M = L // block
        table = torch.randperm(B * M, generator=g).int().reshape(B, M)
        pools = []
        for t in store:
            pool = torch.zeros(B * M, block, t.shape[-1], dtype=t.dtype)
            pool[table.long().flatten()] = t.reshape(B * M, block, -1)
            pools.append(pool)
        store, table = pools, table.cuda()
    store = [t.unsqueeze(2).contiguous().cuda() for t in store] + ([None] if fp8 else [])
    return dict(q=q.cuda(), q_rope=qr.cuda(), kv=store[0], k_rope=store[1], table=table, rows=rows.cuda(),
                both=torch.cat([q, qr], -1).double().cuda())


def call(s, lengths, prefix, **kw):
    return dsa_amd.forward_shared(s["q"], s["kv"], s["q_rope"], s["k_rope"], lengths.int().cuda(), prefix,
                                  block_table=s["table"], **kw)


def check(s, lengths, prefix, scale=1 / 24):
    """The call against the formula."""
    out, top, total = (t.double() for t in call(s, lengths, prefix, scale=scale))
    B, SQ, H, _ = out.shape
    for b in range(B):
        rows = torch.cat([s["rows"][0, :prefix], s["rows"][b, prefix:]])
        for t in range(SQ):
            n = int(lengths[b, t])
            got = out[b, t], top[b, 0, t], total[b, 0, t]
            if n == 0:
                assert not got[0].any() and (got[1] == -INF).all() and not got[2].any()
                continue
            score = (s["both"][b, t][:, None] * rows[:n]).sum(-1) * scale
            peak = score.amax(-1)  # NaN where a score is; with +inf beside it, +inf is returned
            peak[(score == INF).any(-1)] = INF
            w = torch.exp(score - peak[:, None])
            norm = w.sum(-1)
            want = (w[:, :, None] * rows[:n, :512]).sum(1) / norm[:, None]
            size = (w[:, :, None] * rows[:n, :512].abs()).sum(1) / norm[:, None]
            where = f"sequence {b} query {t}"
            assert torch.equal(got[2].isnan(), norm.isnan()), where
            assert torch.equal(got[1].isnan(), peak.isnan()), where
            assert torch.equal(got[1].isinf(), peak.isinf()) and torch.equal(got[1][peak.isinf()], peak[peak.isinf()]), where
            assert torch.equal(got[0].isnan(), want.isnan()), where
            live = ~want.isnan()
            bound = (2.0 ** -8 + 2.0 ** -12) * (size + want.abs()) + 1e-30
            assert ((got[0] - want).abs() <= bound)[live].all(), where
            some = peak.isfinite()
            assert ((got[1] - peak).abs()[some] <= 2.0 ** -14).all(), where
            some = norm.isfinite()
            assert ((got[2] / norm - 1).abs()[some] <= 2.0 ** -12).all(), where


def steps(*ends, queries):
    """Causal lengths of queries that end at these."""
    return torch.tensor(ends)[:, None] - (queries - 1 - torch.arange(queries))


# B, SQ, H: 16, 32, 48, 64 and 128 query rows a block; stacked ones of a prefix and a sequence's own
SHAPES = [(1, 1, 16), (1, 2, 16), (2, 3, 16), (1, 2, 32), (3, 1, 64), (1, 8, 16), (2, 2, 64), (1, 3, 128), (5, 1, 16)]


@pytest.mark.parametrize("layout", ["rows", "paged16", "paged7"])
@pytest.mark.parametrize("value", [INF, -INF])
@pytest.mark.parametrize("B, SQ, H", SHAPES)
def test_a_seen_infinity(B, SQ, H, value, layout):
    """One infinite element of a row: NaN in every column of the heads whose
    product with it is +inf, and in its own column (0 times an infinity) of the
    others, whether or not the tile that it lies in is seen whole."""
    prefix, L = 70, 150
    ends = [149, 131, 97, 71, 128][:B]
    lengths = steps(*ends, queries=SQ)
    last = int(lengths[0, -1]) - 1
    # the first tile, the prefix's last rows and the first behind it, a whole tile, the last tile, the newest row (of the last query only)
    for row, column in zip((3, 64, 69, 70, 75, 100, 127, 128, last - SQ, last), (0, 131, 511, 7, 64, 300, 255, 90, 128, 399)):
        def edit(kv, kr):
            kv[0, row, column] = value
        check(make(B, SQ, H, L, layout, edit, seed=row), lengths, prefix)


@pytest.mark.parametrize("layout", ["rows", "paged7"])
@pytest.mark.parametrize("B, SQ, H", SHAPES)
def test_seen_infinities_do_not_depend_on_other_queries(B, SQ, H, layout):
    """A query's result is the same bits alone, whatever the rest of its block sees."""
    def edit(kv, kr):
        kv[:, 40, 17], kv[:, 100, 300], kv[:, 75, 5] = INF, -INF, NAN

    s = make(B, SQ, H, 150, layout, edit, seed=5)
    for others in (150, 101, 75, 41, 20, 0):
        lengths = torch.full((B, SQ), others)
        lengths[0, 0] = 74
        check(s, lengths, 0)


@pytest.mark.parametrize("layout", ["rows", "paged16"])
@pytest.mark.parametrize("B, SQ, H", [(1, 1, 16), (2, 2, 64), (2, 3, 16)])
def test_a_seen_infinity_in_the_rotary_part(B, SQ, H, layout):
    """No value of the output is infinite there: a score of -inf is a weight of 0."""
    def edit(kv, kr):
        kr[0, 20, 3] = kr[0, 90, 40] = INF

    check(make(B, SQ, H, 130, layout, edit, seed=1), steps(*[128, 111][:B], queries=SQ), 64)


@pytest.mark.parametrize("layout", ["rows", "paged16", "paged7"])
@pytest.mark.parametrize("B, SQ, H", SHAPES)
def test_every_seen_score_infinite(B, SQ, H, layout):
    """-inf in all of them: max -inf and NaN, by the formula, not the zeros of a query that sees nothing."""
    def edit(kv, kr):
        kv[:, :, 7] = INF

    s = make(B, SQ, H, 110, layout, edit, seed=3)
    for ends in ((110, 33, 64, 1, 70), (32, 31, 1, 100, 2)):
        check(s, steps(*ends[:B], queries=SQ).clamp_min(0), 0)
        check(s, steps(*ends[:B], queries=SQ).clamp_min(0), 32)

    def some(kv, kr):  # and later rows finite again
        kv[:, :40, 7] = INF

    check(make(B, SQ, H, 110, layout, some, seed=3), steps(*(110, 33, 64, 41, 70)[:B], queries=SQ).clamp_min(0), 0)


@pytest.mark.parametrize("layout", ["rows", "paged7"])
@pytest.mark.parametrize("B, SQ, H", SHAPES)
def test_a_seen_nan(B, SQ, H, layout):
    def edit(kv, kr):
        kv[0, 5, 9], kv[-1, 80, 200], kr[-1, 81, 2] = NAN, NAN, NAN

    check(make(B, SQ, H, 110, layout, edit, seed=4), steps(*(110, 33, 64, 85, 81)[:B], queries=SQ), 32)
    check(make(B, SQ, H, 110, layout, lambda kv, kr: kv.fill_(NAN), seed=4), steps(*(110, 33, 64, 85, 81)[:B], queries=SQ), 0)


@pytest.mark.parametrize("layout", ["fp8", "fp8_paged16", "fp8_paged7"])
@pytest.mark.parametrize("B, SQ, H", SHAPES)
def test_seen_specials_of_fp8_rows(B, SQ, H, layout):
    """A NaN code; an infinite scale over codes that are 0 but for one; a scale that is NaN."""
    def code(rows):
        rows[0, 5, 300] = 0x7F

    def scale(rows):
        rows[0, 66, :512], rows[-1, 97, :512] = 0, 0
        rows[0, 66, 130], rows[-1, 97, 131] = 0x38, 0xB8
        for b, r, block in ((0, 66, 1), (-1, 97, 2)):
            rows[b, r, 512 + 4 * block:516 + 4 * block].view(torch.float32).fill_(INF)

    def bad_scale(rows):
        rows[-1, 90, 512:516].view(torch.float32).fill_(NAN)

    def alone(rows):  # every code of an infinite block of one sign: +inf or NaN scores but for heads of the other sign
        rows[0, 97, 128:256] = 0x38
        rows[0, 97, 516:520].view(torch.float32).fill_(INF)

    for edit in (code, scale, bad_scale, alone):
        s = make(B, SQ, H, 110, layout, edit, seed=6)
        if edit is alone:  # one head of one sign there: its score is -inf, and the block's 128 columns NaN
            for t in (s["q"], s["both"]):
                t[0, :, 3, 128:256] = -t[0, :, 3, 128:256].abs()
        check(s, steps(*(110, 33, 64, 98, 101)[:B], queries=SQ), 32)
        check(s, steps(*(98, 33, 64, 110, 101)[:B], queries=SQ), 0)


@pytest.mark.parametrize("layout", ["paged7", "fp8", "fp8_paged16", "fp8_paged7"])
@pytest.mark.parametrize("B, SQ, H", [(4, 1, 16), (3, 4, 16), (2, 2, 64), (2, 1, 128)])
def test_unseen_specials(B, SQ, H, layout):
    """Codes, scales and rotary parts of every kind in rows that no query of a sequence sees."""
    P, L = 70, 128
    lengths = steps(*[115, 73, 70, 101][:B], queries=SQ)
    clean = call(make(B, SQ, H, L, layout, lambda *t: None, seed=8), lengths, P)

    def edit(*store):
        g = torch.Generator().manual_seed(0)
        for b in range(B):
            n = max(P, int(lengths[b].max()))
            for t in store:
                hidden = t[b, n:]
                if t.dtype == torch.uint8:
                    hidden.copy_(torch.randint(0, 256, hidden.shape, generator=g, dtype=torch.uint8))
                    hidden[::3, :512] = 0x7F
                    hidden[1::3, 512:528].view(torch.float32).fill_(INF)
                    hidden[2::3, 512:528].view(torch.float32).fill_(NAN)
                else:
                    hidden[::2], hidden[1::2] = INF, NAN
                if b > 0:  # of the prefix only sequence 0's rows count
                    t[b, :P] = 0xFF if t.dtype == torch.uint8 else NAN

    for a, b in zip(clean, call(make(B, SQ, H, L, layout, edit, seed=8), lengths, P)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("layout", ["rows", "paged16", "paged7"])
@pytest.mark.parametrize("rows_a_block", [16, 32, 64, 128])
@pytest.mark.parametrize("sign", [1, -1])
def test_huge_scores(sign, rows_a_block, layout):
    """Scores up to 2^37, exact in 32 bits (one product each, scale 1), more than
    200 apart: all the weight is the largest one's.  The output is its row, the sum
    1 and max the score itself, all exact."""
    L, keys = 140, 131

    def edit(kv, kr):
        kv.mul_(2.0 ** 30)
        # distinct bf16 values, 128 in each power of two
        order = torch.randperm(L, generator=torch.Generator().manual_seed(2))[:kv.shape[1]].double()
        order = torch.cat([order, torch.zeros(kv.shape[1] - order.numel(), dtype=torch.float64)])
        kv[0, :, 0] = (sign * 2.0 ** (36 + order // 128) * (1 + order % 128 / 128)).bfloat16()

    s = make(1, rows_a_block // 16, 16, L, layout, edit, seed=9)
    s["q"].zero_(), s["q_rope"].zero_()
    s["q"][..., 0] = 1
    lengths = torch.full((1, rows_a_block // 16), keys)
    out, top, total = call(s, lengths, 0, scale=1.0)
    score = s["rows"][0, :keys, 0].cpu()
    best = int(score.argmax())
    assert (score == score[best]).sum() == 1
    assert torch.equal(out.double(), s["rows"][0, best, :512].expand(out.shape))
    assert (total == 1).all()
    assert (top.cpu().double() == score[best]).all()
