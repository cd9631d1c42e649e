"""forward_shared in long pieces: planned for one to three compute units, so
that a piece holds ten tiles and more, and with scores that rise far within one
piece, so that it is computed a second time.

Tolerances as in test_gpu_shared.py; a piece here holds fewer than 2048 keys."""
import ctypes
import math

import pytest
import torch

import dsa_amd
from dsa_amd import _lib
from test_gpu_shared import causal, check

pytestmark = pytest.mark.gpu

LAYOUTS = {"rows": (0, False), "paged16": (16, False), "paged7": (7, False), "fp8": (0, True), "fp8_paged16": (16, True),
           "fp8_paged5": (5, True)}


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm GPU")
    torch.cuda.init()


def make(B, SQ, H, P, S, layout, ramp=None, seed=0):
    """``ramp [P + S]``: value 0 of each key row, beside a 40 in every query; rows past it are zeros."""
    block, fp8 = LAYOUTS[layout]
    g = torch.Generator().manual_seed(seed)
    L = P + S if not block else -(-(P + S) // block) * block
    kv, kr = torch.randn(B, L, 512, generator=g).bfloat16(), torch.randn(B, L, 64, generator=g).bfloat16()
    q, qr = torch.randn(B, SQ, H, 512, generator=g).bfloat16(), torch.randn(B, SQ, H, 64, generator=g).bfloat16()
    if ramp is not None:
        q[..., 0], kv[:, :P + S, 0] = 40, ramp.bfloat16()
    kv[:, :P], kr[:, :P] = kv[:1, :P].clone(), kr[:1, :P].clone()
    store = [dsa_amd.quantize_kv_fp8(kv, kr)] if fp8 else [kv, kr]
    if fp8:
        codes = store[0][..., :512].contiguous().view(torch.float8_e4m3fn).double()
        scale = store[0][..., 512:528].contiguous().view(torch.float32).double()
        rows = torch.cat([(codes.unflatten(-1, (4, 128)) * scale[..., None]).flatten(-2), kr.double()], -1)
    else:
        rows = torch.cat([kv, kr], -1).double()
    table = None
    if block:
        M = L // block
        table = torch.randperm(B * M + 2, generator=g)[:B * M].int().reshape(B, M)
        pools = []
        for t in store:
            pool = torch.zeros(B * M + 2, block, t.shape[-1], dtype=t.dtype)
            pool[table.long().flatten()] = t.reshape(B * M, block, -1)
            pools.append(pool)
        store, table = pools, table.cuda()
    store = [t.unsqueeze(2).contiguous().cuda() for t in store] + ([None] if fp8 else [])
    return dict(q=q.cuda(), q_rope=qr.cuda(), kv=store[0], k_rope=store[1], rows=rows.cuda(), table=table, P=P, L=L,
                block=block)


def run(s, lengths, cus, prefix):
    """The C entry, planned for ``cus`` compute units."""
    lib, a = _lib.load(), _lib.DsaSharedArgs()
    B, SQ, H, _ = s["q"].shape
    out = torch.full_like(s["q"], math.nan)
    top = torch.full((B, 1, SQ, H), math.nan, device="cuda")
    total = torch.full_like(top, math.nan)
    a.q, a.kv, a.q_rope, a.lengths = (t.data_ptr() for t in (s["q"], s["kv"], s["q_rope"], lengths))
    a.k_rope = None if s["k_rope"] is None else s["k_rope"].data_ptr()
    a.kv_format = _lib.KV_FP8 if s["k_rope"] is None else _lib.KV_BF16
    a.out, a.out_max, a.out_sum = out.data_ptr(), top.data_ptr(), total.data_ptr()
    a.B, a.SQ, a.H, a.L, a.prefix, a.num_cus = B, SQ, H, s["L"], prefix, cus
    if s["table"] is not None:
        a.block_table, a.max_blocks = s["table"].data_ptr(), s["table"].shape[1]
        a.block_size, a.num_blocks = s["kv"].shape[1], s["kv"].shape[0]
    a.workspace_bytes = lib.dsa_fwd_shared_ws_bytes(ctypes.byref(a))
    assert a.workspace_bytes > 0
    workspace = torch.full((a.workspace_bytes,), 255, device="cuda", dtype=torch.uint8)  # NaN, where read before written
    a.workspace = workspace.data_ptr()
    rc = lib.dsa_fwd_shared(ctypes.byref(a), torch.cuda.current_stream().cuda_stream)
    assert rc == 0, lib.dsa_last_error()
    torch.cuda.synchronize()
    return out, top, total


# (B, SQ, H): blocks of 16, 32, 48, 64, 96 and 128 rows, and stacked ones of a prefix
ROWS = [(1, 1, 16), (1, 2, 16), (1, 1, 48), (1, 4, 16), (1, 1, 96), (1, 1, 128), (3, 1, 16), (2, 3, 16), (5, 2, 16), (2, 1, 128)]


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("B, SQ, H", ROWS)
def test_long_pieces(B, SQ, H, layout):
    """Ten to forty tiles a piece, odd and even numbers of them, the end anywhere in a tile."""
    for keys, cus in ((320, 1), (352, 1), (345, 2), (371, 1), (1285, 3)):
        P = 0 if B == 1 else keys // 2 + 5
        s = make(B, SQ, H, P, keys - P, layout, seed=keys)
        ends = torch.tensor([keys, keys - 40, keys - 1, P + 1, keys - 33])[:B]
        lengths = causal(B, SQ, ends)
        print(layout, B, SQ, H, keys, cus, flush=True)
        check(run(s, lengths, cus, P), s, lengths)
        if P:  # the same rows, nothing shared
            check(run(s, lengths, cus, 0), s, lengths)


@pytest.mark.parametrize("layout", [k for k, v in LAYOUTS.items() if v[0]])
@pytest.mark.parametrize("B, SQ, H", ROWS)
def test_bad_entries_late_in_a_long_piece(B, SQ, H, layout):
    """Entries outside the pool in the last tiles of a piece of a dozen, in the middle, and in its first."""
    keys = 371
    P = 0 if B == 1 else 200
    for bad in ((360,), (0,), (180, 190), (31, 300, 370), (192, 224, 256)):
        s = make(B, SQ, H, P, keys - P, layout, seed=7)
        live = torch.ones(B, s["L"], dtype=torch.bool, device="cuda")
        for key in bad:
            entry = key // s["block"]
            s["table"][0, entry] = (-1, s["kv"].shape[0], (1 << 31) - 1)[key % 3]
            rows = torch.arange(s["L"], device="cuda") // s["block"] == entry
            live[0, rows] = False
            live[:, rows & (torch.arange(s["L"], device="cuda") < P)] = False
        lengths = causal(B, SQ, torch.tensor([keys, keys - 40, keys - 1, P + 1, keys - 33])[:B])
        print(layout, B, SQ, H, bad, flush=True)
        check(run(s, lengths, 1, P), s, lengths, live=live)


@pytest.mark.parametrize("bad", [False, True])
@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("B, SQ, H", ROWS)
def test_scores_that_rise_within_a_piece(B, SQ, H, layout, bad):
    """Weights that grow from 2^-140 to 1 along one piece: its first reference
    is passed by more than 2^64, and the piece is computed once more.  A block
    of each, with an entry outside the pool in the middle."""
    if bad and not LAYOUTS[layout][0]:
        pytest.skip("no block table")
    keys = 363
    P = 0 if B == 1 else 330  # stacked: the prefix is a piece of its own
    # product 0 of a score: 40 x (-30 .. 30) / 24 = -50 .. 50, 72 to either side in log2 units
    for sign in (1, -1):
        s = make(B, SQ, H, P, keys - P, layout, ramp=torch.linspace(-30 * sign, 30 * sign, keys), seed=3)
        live = None
        if bad:
            entry = 170 // s["block"]
            s["table"][:, entry] = -1
            live = (torch.arange(s["L"], device="cuda") // s["block"] != entry).expand(B, -1)
        lengths = causal(B, SQ, torch.tensor([keys, keys - 9, keys - 1, keys - 20, keys - 12])[:B])
        # one workgroup: each item is one piece.  Its first two tiles (either group's first) against all of it
        q = torch.cat([s["q"], s["q_rope"]], -1).double()[0, -1]
        score = q @ s["rows"][0, :P or keys].t() / 24 * math.log2(math.e)
        rise = score.amax(-1) - score[:, :64].amax(-1)
        assert (rise > 66).all() if sign > 0 else (rise < 1).all()
        print(layout, B, SQ, H, sign, flush=True)
        # a score holds a product up to 1200 beside the 480: 3.5 times the errors
        check(run(s, lengths, 1, P), s, lengths, live=live, sharp=3.5)
        check(run(s, lengths, 2, P), s, lengths, live=live, sharp=3.5)
