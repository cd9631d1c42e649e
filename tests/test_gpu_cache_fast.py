"""The host fast path of the paged cache's operators (dsa_amd/_fast_cache*.so,
built from csrc/fast_cache.cpp): the same results as the Python path, and None
for whatever that refuses or does besides."""
import sys

import pytest
import torch

import dsa_amd
from dsa_amd import api, paging

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def fast():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm GPU")
    module = api._fast_cache()
    assert module is not None, "the fast path module is built by dsa_amd.build"
    return module


def i32(*v):
    return torch.tensor(v, dtype=torch.int32).cuda()


def table_args():
    return [i32(*range(12)).view(3, 4), i32(5, 0, 16), i32(3, 9, 0), i32(40, 41, 42, 43), 4, 14]


def rotary_args(dim=3, out=False):
    x = torch.randn((2, 5, 4, 96)[4 - dim:]).bfloat16().cuda()
    positions = torch.arange(x.shape[:-2].numel()).view(x.shape[:-2]).cuda()
    return [x, positions, dsa_amd.rotary_frequencies(64).cuda(), True, 32, False, 1.5, torch.empty_like(x) if out else None]


def write_args(fp8=False, turned=True):
    kv = torch.randn(5, 576).bfloat16().cuda()
    where = [torch.arange(5).cuda(), dsa_amd.rotary_frequencies(64).cuda()] if turned else [None, None]
    cache = ([torch.zeros(3, 4, 656, dtype=torch.uint8).cuda(), None] if fp8 else
             [torch.zeros(3, 4, 512).bfloat16().cuda(), torch.zeros(3, 4, 64).bfloat16().cuda()])
    return [kv[:, :512], kv[:, 512:], i32(3, -1, 11, 12, 0), *cache, *where, False, 1.0, True]


def shared_args(layout="paged"):
    bf = lambda *shape: torch.randn(shape, generator=torch.Generator().manual_seed(len(shape))).bfloat16().cuda()  # noqa: E731
    q, kv, qr, kr = bf(2, 3, 16, 512), bf(6, 16, 1, 512), bf(2, 3, 16, 64), bf(6, 16, 1, 64)
    lengths, table = i32(40, 41, 42, 7, 8, 9).view(2, 3), i32(0, 1, 2, 0, 4, 5).view(2, 3)
    if layout == "rows":
        return [q, kv.view(2, 48, 1, 512), qr, kr.view(2, 48, 1, 64), lengths, 0, None, None]
    if layout == "fp8":
        return [q, dsa_amd.quantize_kv_fp8(kv, kr), qr, None, lengths, 16, 0.05, table]
    return [q, kv, qr, kr, lengths, 16, 192 ** -0.5, table]


def test_taken_and_equal(fast, monkeypatch):
    module = sys.modules["dsa_amd.rotary"]
    for args in (rotary_args(), rotary_args(4), rotary_args(4, out=True)):
        taken = fast.rotary(*args)
        assert taken is not None and (args[7] is None or taken is args[7])
        taken = taken.clone()
        monkeypatch.setattr(module, "_fast_cache", lambda: None)
        kw = dict(interleaved=args[3], start=args[4], transposed=args[5], magnitude=args[6], out=args[7])
        assert torch.equal(dsa_amd.rotary(*args[:3], **kw), taken)
        monkeypatch.undo()
        assert torch.equal(dsa_amd.rotary(*args[:3], **kw), taken)
    one, two = table_args(), table_args()
    taken = fast.extend_block_table(*one)
    monkeypatch.setattr(paging, "_fast_cache", lambda: None)
    for a, b in zip(taken, dsa_amd.extend_block_table(*two)):
        assert a.dtype == b.dtype and torch.equal(a, b)
    assert torch.equal(one[0], two[0])
    for args in (write_args(), write_args(True), write_args(turned=False)):
        assert fast.write_kv_rows(*args) == 0
        again = [a.clone() if i in (3, 4) and a is not None else a for i, a in enumerate(args)]
        for i in (3, 4):
            if again[i] is not None:
                again[i].zero_()
        dsa_amd.write_kv_rows(*again[:5], positions=again[5], frequencies=again[6], interleaved=again[7],
                              magnitude=again[8], pow2_scales=again[9])
        assert torch.equal(args[3], again[3]) and (args[4] is None or torch.equal(args[4], again[4]))


@pytest.mark.parametrize("layout", ["rows", "paged", "fp8"])
def test_attention_taken_and_equal(fast, monkeypatch, layout):
    args = shared_args(layout)
    taken = fast.forward_shared(*args)
    assert taken is not None
    monkeypatch.setattr(sys.modules["dsa_amd.shared"], "_fast_cache", lambda: None)
    for a, b in zip(taken, dsa_amd.forward_shared(*args[:6], scale=args[6], block_table=args[7])):
        assert a.shape == b.shape and a.dtype == b.dtype and torch.equal(a, b)


@pytest.mark.parametrize("call, make, bad", [
    ("forward_shared", shared_args, {
        0: [None, "cpu", "float", "short", "last", "empty", "unaligned"], 1: [None, "cpu", "float", "bytes", "unaligned"],
        2: [None, "cpu", "float", "short", "last", "unaligned"], 3: [None, "cpu", "float", "short", "unaligned"],
        4: [None, "cpu", "long", "short", "last"], 5: [-1, 49, 1.0, True, None], 6: [0.0, -1.0, float("nan"), float("inf"), 1, "x"],
        7: [3, "cpu", "long", "short", "last"]}),
    ("extend_block_table", table_args, {
        0: [None, torch.zeros(12).int(), "cpu", "long", "apart", torch.zeros(4, 0).int()], 1: ["cpu", "long", "short"],
        2: ["cpu", "long", "short"], 3: ["cpu", "long", "apart"], 4: [0, -1, 2 ** 31, 4.0, True, None],
        5: [-1, 2 ** 31, 2.0, False]}),
    ("rotary", rotary_args, {
        0: [None, 3, "cpu", "long", "last", "grad", "empty", torch.zeros(2, 2)], 1: [None, "cpu", "float", "short", "apart"],
        2: [None, "cpu", "float", "apart", torch.zeros(0).double()], 3: [None, 1], 4: [-1, 33, 1.0, True], 5: [None, 0],
        6: [float("nan"), float("inf"), 1e39, None, 1], 7: [3, "cpu", "short", "over"]}),
    ("write_kv_rows", write_args, {
        0: [None, "cpu", "float", "short", "last", "empty", "odd"], 1: [None, "cpu", "float", "short", "last"],
        2: [None, "cpu", "long", "short", "apart"], 3: [None, "cpu", "float", "last", "bytes"],
        4: [None, "cpu", "float", "short"], 5: [None, "cpu", "float", "short"], 6: [None, "cpu", "float", "short"],
        7: [None, 1], 8: [float("nan"), None, 1, 1e39], 9: [None, 0]})])
def test_declines(fast, call, make, bad):
    """Declined before anything is allocated or written."""
    how = {"cpu": lambda t: t.cpu(), "long": lambda t: t.long(), "float": lambda t: t.float(), "short": lambda t: t[:-1],
           "apart": lambda t: torch.stack([t, t], -1)[..., 0], "last": lambda t: t.transpose(-1, -2),
           "grad": lambda t: t.clone().requires_grad_(), "empty": lambda t: t[:0], "bytes": lambda t: t.byte(),
           "unaligned": lambda t: torch.cat([t.flatten()[:1], t.flatten()])[1:].view(t.shape),
           "odd": lambda t: torch.zeros(5, 577).bfloat16().cuda()[:, :512]}
    for at, values in bad.items():
        for value in values:
            args = make()
            if isinstance(value, str) and value == "over":
                args[7] = torch.zeros(args[0].numel() + 8).bfloat16().cuda()
                args[0], args[7] = args[7][:-8].view(make()[0].shape), args[7][8:].view(make()[0].shape)
            elif isinstance(value, str) and value in how:
                args[at] = how[value](args[at] if args[at] is not None else torch.empty_like(args[0]))
            else:
                args[at] = value
            kept = [a.clone() if isinstance(a, torch.Tensor) else a for a in args]
            torch.cuda.synchronize()
            before = torch.cuda.memory_allocated()
            print(call, at, value, flush=True)
            assert getattr(fast, call)(*args) is None, (at, value)
            torch.cuda.synchronize()
            assert torch.cuda.memory_allocated() == before
            for a, k in zip(args, kept):
                assert not isinstance(a, torch.Tensor) or torch.equal(a, k)


def test_a_gradient_is_recorded_all_the_same(fast):
    x, positions, freq = rotary_args()[:3]
    x.requires_grad_()
    y = dsa_amd.rotary(x, positions, freq)
    y.sum().backward()
    assert x.grad is not None
    with torch.no_grad():
        assert torch.equal(dsa_amd.rotary(x, positions, freq), y)


@pytest.mark.parametrize("quick", [True, False])
def test_autograd_is_told_of_writes(fast, monkeypatch, quick):
    """A product that saved a cache for its gradient refuses once the cache has been written."""
    if not quick:
        for name in ("rotary", "paging"):
            monkeypatch.setattr(sys.modules["dsa_amd." + name], "_fast_cache", lambda: None)
    args = write_args()
    w = torch.ones(512, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    y = (args[3] * w).sum()
    dsa_amd.write_kv_rows(*args[:5])
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    for t in args[3:5]:
        with pytest.raises(ValueError, match="gradient"):
            dsa_amd.write_kv_rows(*args[:3], *(c.clone().requires_grad_() if c is t else c for c in args[3:5]))
    x, positions, freq = rotary_args()[:3]
    before = x._version
    dsa_amd.rotary(x, positions, freq, out=x)
    assert x._version == before + 1
    table = table_args()
    dsa_amd.extend_block_table(*table)
    assert table[0]._version == 1 + i32(*range(12)).view(3, 4)._version
    with torch.inference_mode():
        x, positions, freq = rotary_args()[:3]
        dsa_amd.rotary(x, positions, freq, out=x)
        dsa_amd.write_kv_rows(*write_args()[:5])
    dsa_amd.rotary(x, positions, freq, out=x)
