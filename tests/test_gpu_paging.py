"""Block tables, slot maps and cache row writes against plain host code (whole
numbers and copied bits: equal, not near)."""
import pytest
import torch

import dsa_amd

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm GPU")
    torch.cuda.init()


# ------------------------------------------------------------ block tables

def host_extend(table, lengths, new, free, block, most):
    """The step, token by token, in plain Python."""
    table = [row[:] for row in table]
    width, taken, slots, positions, starts, totals = len(table[0]), 0, [], [], [0], []
    for row, held, add in zip(table, lengths, new):
        held, add = max(held, 0), max(add, 0)
        for column in range(-(-held // block), min(-(-(held + add) // block), width)):
            row[column] = free[taken] if taken < len(free) else -1
            taken += 1
        for at in range(held, held + add):
            entry = row[at // block] if at // block < width else -1
            slots.append(entry * block + at % block if entry >= 0 else -1)
            positions.append(at)
        starts.append(starts[-1] + add)
        totals.append(held + add)
    pad = max(0, most - len(slots))
    return table, (slots + [-1] * pad)[:most], (positions + [0] * pad)[:most], starts, totals, [taken]


def run_extend(table, lengths, new, free, block, most):
    i32 = lambda v: torch.tensor(v, dtype=torch.int32).cuda()  # noqa: E731
    t = i32(table)
    return [t] + list(dsa_amd.extend_block_table(t, i32(lengths), i32(new), i32(free), block, most))


def check_extend(table, lengths, new, free, block, most):
    got = run_extend(table, lengths, new, free, block, most)
    want = host_extend(table, lengths, new, free, block, most)
    for g, w, name in zip(got, want, ("table", "slots", "positions", "starts", "totals", "used")):
        assert g.tolist() == w, name


def scene(batch, block, width, held, add, seed):
    g = torch.Generator().manual_seed(seed)
    rnd = lambda high: torch.randint(0, high + 1, (batch,), generator=g).tolist()  # noqa: E731
    lengths, new = rnd(held), rnd(add)
    order = torch.randperm(batch * width, generator=g).tolist()
    table = [[order[b * width + c] if c < -(-lengths[b] // block) else -1 for c in range(width)] for b in range(batch)]
    used = {e for row in table for e in row}
    return table, lengths, new, [e for e in order if e not in used], block, sum(new)


@pytest.mark.parametrize("batch, block, width, held, add", [
    (1, 64, 4, 0, 1), (1, 1, 9, 4, 5), (3, 16, 8, 64, 60), (64, 64, 40, 2400, 1), (257, 16, 12, 150, 3),
    (1000, 48, 5, 200, 4), (4096, 16, 3, 40, 2), (5, 7, 400, 1000, 1700), (48, 16, 130, 0, 2047)])
def test_extend(batch, block, width, held, add):
    check_extend(*scene(batch, block, width, held, add, batch + block))


def test_extend_at_borders():
    table = [[3, -1, -1], [4, 5, -1], [6, 7, 8], [-1, -1, -1]]
    # a full block, one short of full, a full row, an empty sequence; padding behind
    check_extend(table, [4, 7, 12, 0], [1, 1, 0, 4], [20, 21, 22], 4, 9)
    # nothing new at all
    check_extend(table, [4, 7, 12, 0], [0, 0, 0, 0], [20], 4, 3)
    check_extend(table, [4, 7, 12, 0], [0, 0, 0, 0], [], 4, 0)
    # the list runs short inside a sequence; the rest get -1
    check_extend(table, [4, 7, 12, 0], [5, 3, 0, 6], [20, 21], 4, 14)
    check_extend(table, [4, 7, 12, 0], [5, 3, 0, 6], [], 4, 14)
    # rows too narrow: blocks past the row are not taken
    check_extend(table, [4, 7, 12, 0], [20, 3, 2, 13], [20, 21, 22, 23, 24, 25, 26], 4, 38)
    # more tokens than the outputs hold
    check_extend(table, [4, 7, 12, 0], [5, 3, 0, 6], [20, 21, 22, 23, 24, 25, 26], 4, 5)
    # negative counts are none, and a partly filled block without an entry has no slots
    check_extend(table, [-3, 6, 12, 2], [2, -5, 0, 1], [20, 21], 4, 4)


def test_extend_saturates():
    """Counts whose sums pass 2^31 - 1 stay there; nothing is written past the outputs."""
    big = (1 << 31) - 1
    table, slots, positions, starts, totals, used = run_extend([[1, 2], [3, 4], [5, 6]], [0, 0, 5], [big, big, 1],
                                                               [10, 11, 12, 13, 14], 8, 20)
    assert starts.tolist() == [0, big, big, big] and totals.tolist() == [big, big, 6] and used.tolist() == [4]
    assert table.tolist() == [[10, 11], [12, 13], [5, 6]]
    assert slots.tolist() == [80 + i for i in range(16)] + [-1] * 4 and positions.tolist() == list(range(20))


def test_extend_slot_past_31_bits():
    """A row number past 2^31 - 1 is no slot."""
    big = (1 << 31) - 1
    _, slots, _, _, _, _ = run_extend([[big // 8, big // 8 + 1]], [6], [4], [], 8, 4)
    assert slots.tolist() == [big // 8 * 8 + 6, big // 8 * 8 + 7, -1, -1]


def test_extend_step_by_step_equals_at_once():
    table, lengths, new, free, block, _ = scene(20, 16, 30, 200, 0, 5)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32).cuda()  # noqa: E731
    add = torch.randint(0, 40, (20,), generator=torch.Generator().manual_seed(1)).int().cuda()
    once, steps, held, left = i32(table), i32(table), i32(lengths), i32(free)
    at_once = dsa_amd.extend_block_table(once, held, add, left, block, int(add.sum()))
    where = {}
    for k in range(40):
        step = (add > k).int()
        s = dsa_amd.extend_block_table(steps, held, step, left, block, 20)
        n = int(step.sum())
        where.update({(b, p): r for b, p, r in zip(torch.nonzero(step).flatten().tolist(), s[1][:n].tolist(),
                                                   s[0][:n].tolist())})
        held, left = s[3], left[int(s[4]):].contiguous()
    assert held.tolist() == at_once[3].tolist()
    # the same number of blocks, each row of the cache used once
    assert (steps >= 0).sum() == (once >= 0).sum()
    assert len(set(where.values())) == len(where) == int(add.sum()) and -1 not in where.values()


def test_extend_refusals():
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")  # noqa: E731
    good = [i32(2, 4), i32(2), i32(2), i32(5), 16, 4]
    dsa_amd.extend_block_table(*good)
    for at, value in [(0, i32(2, 4).long()), (0, i32(4, 2).t()), (1, i32(3)), (1, i32(2).long()), (1, i32(2).cpu()),
                      (2, i32(4)[::2]), (2, i32(2, 1)), (3, i32(5).float()), (3, i32(10)[::2]), (4, -16), (5, -1), (5, 1.5)]:
        args = list(good)
        args[at] = value
        with pytest.raises(ValueError):
            dsa_amd.extend_block_table(*args)


# ------------------------------------------------------------ row writes

def rows_for(tokens, seed=0):
    g = torch.Generator().manual_seed(seed)
    proj = torch.randn(tokens, 576, generator=g).bfloat16().cuda()
    kv = (torch.randn(tokens, 512, generator=g) * torch.exp(torch.randn(512, generator=g))).bfloat16().cuda()
    return kv, proj[:, 512:]


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("interleaved", [True, False, None])  # None: not turned
@pytest.mark.parametrize("tokens", [1, 2, 3, 33, 700, 20001])
def test_write(tokens, interleaved, fp8):
    """The rows hold the bits of rotary() and quantize_kv_fp8(); other rows and tokens without a slot are left alone."""
    kv, rope = rows_for(tokens)
    block, blocks = 16, tokens // 16 + 20
    slots = torch.randperm(blocks * block, generator=torch.Generator().manual_seed(3))[:tokens].int()
    if tokens > 2:
        slots[0], slots[tokens // 2], slots[-1] = -1, blocks * block, -(1 << 31)
    live = (slots >= 0) & (slots < blocks * block)
    slots = slots.cuda()
    positions = torch.randint(0, 1 << 20, (tokens,), generator=torch.Generator().manual_seed(4)).cuda()
    freq = dsa_amd.rotary_frequencies(64, scaling="yarn", factor=4.0).cuda()
    kw, turned = {}, rope
    if interleaved is not None:
        kw = dict(positions=positions, frequencies=freq, interleaved=interleaved, magnitude=1.25)
        turned = dsa_amd.rotary(rope.unsqueeze(1), positions, freq, interleaved=interleaved, magnitude=1.25).squeeze(1)
    at = slots[live.cuda()].long()
    if fp8:
        for pow2 in (True, False):
            cache = torch.randint(0, 255, (blocks, block, 1, 656), dtype=torch.uint8, device="cuda")
            want = cache.clone()
            want.view(-1, 656)[at] = dsa_amd.quantize_kv_fp8(kv, turned.contiguous(), pow2)[live.cuda()]
            assert dsa_amd.write_kv_rows(kv, rope, slots, cache, pow2_scales=pow2, **kw) is None
            assert torch.equal(cache, want)
    else:
        cache = torch.randn(blocks, block, 1, 512, device="cuda").bfloat16()
        rcache = torch.randn(blocks, block, 1, 64, device="cuda").bfloat16()
        want, rwant = cache.clone(), rcache.clone()
        want.view(-1, 512)[at], rwant.view(-1, 64)[at] = kv[live.cuda()], turned[live.cuda()]
        dsa_amd.write_kv_rows(kv, rope, slots, cache, rcache, **kw)
        assert torch.equal(cache, want) and torch.equal(rcache, rwant)


def test_write_special_values():
    """NaN and infinities are copied as they are, and quantized as quantize_kv_fp8 does."""
    kv, rope = rows_for(6)
    kv[0, 3], kv[1, 200], kv[2, 511], kv[3], rope[4, 7] = float("nan"), float("inf"), float("-inf"), 0.0, float("nan")
    slots = torch.arange(6, device="cuda", dtype=torch.int32)
    cache = torch.zeros(8, 1, 512, device="cuda", dtype=torch.bfloat16)
    rcache = torch.zeros(8, 1, 64, device="cuda", dtype=torch.bfloat16)
    dsa_amd.write_kv_rows(kv, rope, slots, cache, rcache)
    assert torch.equal(cache[:6, 0].view(torch.int16), kv.view(torch.int16))
    assert torch.equal(rcache[:6, 0].view(torch.int16), rope.contiguous().view(torch.int16))
    rows = torch.zeros(8, 656, device="cuda", dtype=torch.uint8)
    dsa_amd.write_kv_rows(kv, rope, slots, rows)
    assert torch.equal(rows[:6], dsa_amd.quantize_kv_fp8(kv, rope.contiguous()))


def test_write_strided_kv_and_empty():
    big = torch.randn(9, 1024, device="cuda").bfloat16()
    kv, rope = big[::2, 512:], big[::2, 64:128]
    slots = torch.tensor([4, 0, 2, 1, 3], dtype=torch.int32, device="cuda")
    cache = torch.zeros(5, 512, device="cuda", dtype=torch.bfloat16)
    rcache = torch.zeros(5, 64, device="cuda", dtype=torch.bfloat16)
    dsa_amd.write_kv_rows(kv, rope, slots, cache, rcache)
    assert torch.equal(cache[slots.long()], kv) and torch.equal(rcache[slots.long()], rope)
    dsa_amd.write_kv_rows(kv[:0], rope[:0], slots[:0], cache, rcache)
    assert torch.equal(cache[slots.long()], kv)


@pytest.mark.parametrize("fp8", [False, True])
def test_write_far_rows(fp8):
    """Rows past 2^31 elements and 4 GiB of the cache."""
    rows = (1 << 32) // 656 + 64 if fp8 else (1 << 31) // 512 + 64
    kv, rope = rows_for(5)
    slots = torch.tensor([rows - 1, 0, rows // 2 + 9, rows - 30, rows], dtype=torch.int32).cuda()
    at = slots[:4].long()
    if fp8:
        cache = torch.zeros(rows, 656, dtype=torch.uint8, device="cuda")
        dsa_amd.write_kv_rows(kv, rope, slots, cache)
        assert torch.equal(cache[at], dsa_amd.quantize_kv_fp8(kv, rope.contiguous())[:4])
        cache[at] = 0
        assert not cache.view(torch.int64).any()
    else:
        cache = torch.zeros(rows, 512, dtype=torch.bfloat16, device="cuda")
        rcache = torch.zeros(rows, 64, dtype=torch.bfloat16, device="cuda")
        dsa_amd.write_kv_rows(kv, rope, slots, cache, rcache)
        assert torch.equal(cache[at], kv[:4]) and torch.equal(rcache[at], rope[:4])
        cache[at] = 0
        assert not cache.any()


def test_write_the_same_row_twice():
    """The row holds one of the two tokens; the other rows are right."""
    kv, rope = rows_for(64, 8)
    slots = (torch.arange(64, device="cuda") // 2).int()
    cache = torch.zeros(40, 512, device="cuda", dtype=torch.bfloat16)
    rcache = torch.zeros(40, 64, device="cuda", dtype=torch.bfloat16)
    dsa_amd.write_kv_rows(kv, rope, slots, cache, rcache)
    for r in range(32):
        assert torch.equal(cache[r], kv[2 * r]) or torch.equal(cache[r], kv[2 * r + 1])
    assert not cache[32:].any() and not rcache[32:].any()


def test_write_refusals():
    kv, rope = rows_for(4)
    slots = torch.arange(4, device="cuda", dtype=torch.int32)
    cache = torch.zeros(8, 1, 512, device="cuda", dtype=torch.bfloat16)
    rcache = torch.zeros(8, 1, 64, device="cuda", dtype=torch.bfloat16)
    f, p = dsa_amd.rotary_frequencies(64).cuda(), torch.arange(4, device="cuda")
    wide = torch.zeros(4, 1025, device="cuda", dtype=torch.bfloat16)
    bad = [dict(kv=kv.float()), dict(k_rope=rope.half()), dict(kv=kv.cpu()), dict(slots=slots.long()), dict(slots=slots[:3]),
           dict(slots=torch.arange(8, device="cuda", dtype=torch.int32)[::2]), dict(kv_cache=cache.transpose(0, 1)),
           dict(kv_cache=cache.float()), dict(rope_cache=rcache.float()), dict(rope_cache=None), dict(kv=wide[:, 1:513]),
           dict(kv=wide[:, :512]), dict(k_rope=wide[:, 1:65]), dict(positions=p), dict(frequencies=f),
           dict(positions=p[:3], frequencies=f), dict(positions=p, frequencies=f[:16]),
           dict(positions=p.float(), frequencies=f), dict(positions=p, frequencies=f, magnitude=float("nan"))]
    for kw in bad:
        with pytest.raises(ValueError):
            dsa_amd.write_kv_rows(**{**dict(kv=kv, k_rope=rope, slots=slots, kv_cache=cache, rope_cache=rcache), **kw})
    assert not cache.any() and not rcache.any()


# ------------------------------------------------------------ streams and graphs

@pytest.mark.parametrize("fp8", [False, True])
def test_a_captured_step(fp8):
    """Tables, slots and rows of a step in a graph: every replay follows the inputs and equals the eager calls."""
    block, width, batch = 16, 12, 6
    g = torch.Generator().manual_seed(2)
    table = torch.randperm(batch * width, generator=g).int().reshape(batch, width).cuda()
    free = (torch.randperm(20, generator=g) + batch * width).int().cuda()
    lengths, new = torch.zeros(batch, dtype=torch.int32).cuda(), torch.ones(batch, dtype=torch.int32).cuda()
    kv, rope = rows_for(4 * batch)
    f = dsa_amd.rotary_frequencies(64).cuda()
    rows = batch * width + 20

    def caches():
        if fp8:
            return (torch.zeros(rows, block, 1, 656, dtype=torch.uint8, device="cuda"),)
        return (torch.zeros(rows, block, 1, 512, dtype=torch.bfloat16, device="cuda"),
                torch.zeros(rows, block, 1, 64, dtype=torch.bfloat16, device="cuda"))

    def step(table, pools):
        slots, positions, starts, totals, used = dsa_amd.extend_block_table(table, lengths, new, free, block, 4 * batch)
        dsa_amd.write_kv_rows(kv, rope, slots, *pools, positions=positions, frequencies=f)
        return slots, positions, starts, totals, used

    start, pools = table.clone(), caches()
    step(table, pools)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(table, pools)
    for k in range(4):
        lengths.copy_(torch.randint(0, 150, (batch,), generator=g))
        new.copy_(torch.randint(0, 5, (batch,), generator=g))
        kv.copy_(rows_for(4 * batch, seed=k)[0])
        table.copy_(start)
        for t in pools:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        other, others = start.clone(), caches()
        for a, b in zip(got, step(other, others)):
            assert torch.equal(a, b)
        assert torch.equal(table, other) and all(torch.equal(a, b) for a, b in zip(pools, others))
