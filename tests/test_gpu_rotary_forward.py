"""Forward-mode derivatives of rotary and of the operators around it, and
derivatives that they do not have."""
import sys

import pytest
import torch
import torch.autograd.forward_ad as fw

import dsa_amd

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm GPU")
    torch.cuda.init()


@pytest.fixture(params=[True, False], ids=["fast", "python"])
def host(request, monkeypatch):
    if not request.param:
        for name in ("rotary", "paging"):
            monkeypatch.setattr(sys.modules["dsa_amd." + name], "_fast_cache", lambda: None)
    return request.param


def make(shape, dtype=torch.float32, seed=0):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


def inputs(shape, dtype=torch.float32):
    positions = torch.arange(torch.Size(shape[:-2]).numel()).view(shape[:-2]).cuda() * 77
    return make(shape, dtype), make(shape, dtype, 1), positions, dsa_amd.rotary_frequencies(64).cuda()


@pytest.mark.parametrize("transposed", [False, True])
@pytest.mark.parametrize("leaf", [False, True])
@pytest.mark.parametrize("shape, dtype", [((5, 3, 96), torch.float32), ((2, 4, 3, 96), torch.bfloat16)])
def test_tangent(host, shape, dtype, leaf, transposed):
    """The operator is linear in x: its tangent is the same turn of x's, bit for bit."""
    x, t, positions, freq = inputs(shape, dtype)
    kw = dict(interleaved=False, start=16, transposed=transposed, magnitude=0.75)
    with torch.no_grad():
        want, turned = dsa_amd.rotary(x, positions, freq, **kw), dsa_amd.rotary(t, positions, freq, **kw)
    x.requires_grad_(leaf)
    with fw.dual_level():
        y = dsa_amd.rotary(fw.make_dual(x, t), positions, freq, **kw)
        primal, tangent = fw.unpack_dual(y)
        assert tangent is not None and torch.equal(tangent, turned) and torch.equal(primal, want)
        assert fw.unpack_dual(dsa_amd.rotary(x, positions, freq, **kw)).tangent is None
        # a tangent whose last stride is not 1
        apart = torch.stack([t, t], -1)[..., 0]
        y = dsa_amd.rotary(fw.make_dual(x, apart), positions, freq, **kw)
        assert torch.equal(fw.unpack_dual(y).tangent, turned)
        if leaf:  # the gradient beside the tangent
            y.backward(t)
            with torch.no_grad():
                assert torch.equal(x.grad, dsa_amd.rotary(t, positions, freq, **{**kw, "transposed": not transposed}))


def test_function_transforms_are_refused(host):
    """torch.func's stand-ins for tensors: an error, not a derivative of zero."""
    x, t, positions, freq = inputs((5, 3, 64))
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda v: dsa_amd.rotary(v, positions, freq), (x,), (t,))
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda v: dsa_amd.rotary(v, positions, freq).sum())(x)
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda p: dsa_amd.rotary(x, p, freq))(positions.expand(2, 5))


def test_second_derivative(host):
    x, t, positions, freq = inputs((5, 3, 64))
    x.requires_grad_()
    y = dsa_amd.rotary(x, positions, freq)
    g, = torch.autograd.grad((y * y).sum() / 2, x, create_graph=True)
    h, = torch.autograd.grad((g * t).sum(), x)
    with torch.no_grad():  # halves and doubles are exact
        assert torch.equal(g, dsa_amd.rotary(y, positions, freq, transposed=True))
        assert torch.equal(h, dsa_amd.rotary(dsa_amd.rotary(t, positions, freq), positions, freq, transposed=True))


def test_no_tangent_into_out(host):
    x, t, positions, freq = inputs((5, 3, 64))
    with fw.dual_level():
        dual = fw.make_dual(x, t)
        for a, out in ((dual, torch.empty_like(x)), (dual, dual), (x, fw.make_dual(torch.empty_like(x), t))):
            with pytest.raises(ValueError, match="gradient"):
                dsa_amd.rotary(a, positions, freq, out=out)
        with torch.no_grad(), pytest.raises(ValueError, match="gradient"):
            dsa_amd.rotary(dual, positions, freq, out=torch.empty_like(x))
    assert torch.equal(x, make((5, 3, 64)))


def test_frequencies_have_no_gradient(host):
    """Asked for one, the call refuses; it does not return a zero."""
    x, t, positions, freq = inputs((5, 3, 64))
    wanted = freq.clone().requires_grad_()
    for kw in ({}, dict(out=torch.empty_like(x))):
        with pytest.raises(ValueError, match="frequencies"):
            dsa_amd.rotary(x, positions, wanted, **kw)
    with pytest.raises(ValueError, match="frequencies"):
        dsa_amd.rotary(x.clone().requires_grad_(), positions, wanted)
    with torch.no_grad():
        assert torch.equal(dsa_amd.rotary(x, positions, wanted), dsa_amd.rotary(x, positions, freq))
    with fw.dual_level(), pytest.raises(ValueError, match="frequencies"):
        dsa_amd.rotary(x, positions, fw.make_dual(freq, torch.ones_like(freq)))


def test_caches_have_no_tangent(host):
    """A cache that carries a tangent would keep the old one over its new rows."""
    bf16 = lambda *s: torch.randn(s, generator=torch.Generator().manual_seed(0)).bfloat16().cuda()  # noqa: E731
    kv, rope, cache, rcache = bf16(3, 512), bf16(3, 64), bf16(8, 512), bf16(8, 64)
    slots = torch.tensor([1, 4, 6], dtype=torch.int32).cuda()
    kept = cache.clone(), rcache.clone()
    with fw.dual_level():
        dual = [fw.make_dual(c, torch.ones_like(c)) for c in (cache, rcache)]
        for pair in ((dual[0], rcache), (cache, dual[1])):
            with torch.no_grad(), pytest.raises(ValueError, match="gradient"):
                dsa_amd.write_kv_rows(kv, rope, slots, *pair)
            with pytest.raises(ValueError, match="gradient"):
                dsa_amd.write_kv_rows(kv, rope, slots, *pair)
    assert torch.equal(cache, kept[0]) and torch.equal(rcache, kept[1])
