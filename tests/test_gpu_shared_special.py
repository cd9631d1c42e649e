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
            peak = score.amax(-1)
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


