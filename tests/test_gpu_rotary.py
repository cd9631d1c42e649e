"""Rotary positions against complex products in 64 bits.

Tolerance: the angle is exact to 2^-25 of a turn (its 32-bit fraction), 2^-22.3
radians, and the sine and cosine round to 2^-24 or a few of them; each output
is two products and one sum in 32 bits of values up to |x0| + |x1|, so it is
within 2^-21 (|x0| + |x1|) of the exact one before the last rounding (2^-22.3
angle, 2 x 2^-24 for two units in the last place of sine and cosine, 2 x 2^-24
for the magnitude's product and the two products' sum), which adds half a step
of the type, eps / 2 of the value."""
import pytest
import torch

import dsa_amd

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm GPU")
    torch.cuda.init()


def exact(x, positions, freq, interleaved=True, start=0, transposed=False, magnitude=1.0):
    """64-bit result and the sum of the magnitudes that enter each output."""
    x, out = x.double().cpu(), x.double().cpu().clone()
    positions, freq = positions.cpu(), freq.cpu()
    dim, half = 2 * freq.numel(), freq.numel()
    angle = positions.double()[..., None] * freq * (-1 if transposed else 1)
    turn = (torch.polar(torch.ones_like(angle), angle) * magnitude).unsqueeze(-2)
    size = out.abs()
    i0 = start + (torch.arange(0, dim, 2) if interleaved else torch.arange(half))
    i1 = i0 + (1 if interleaved else half)
    z = torch.complex(x[..., i0], x[..., i1]) * turn
    both = (x[..., i0].abs() + x[..., i1].abs()) * abs(magnitude)
    out[..., i0], out[..., i1] = z.real, z.imag
    size[..., i0] = size[..., i1] = both
    return out, size


def check(y, x, positions, freq, **kw):
    ref, size = exact(x, positions, freq, **kw)
    step = torch.finfo(x.dtype).eps / 2
    tiny = torch.finfo(x.dtype).tiny  # below the normal range a step is absolute
    bound = 2.0 ** -21 * size + step * (ref.abs() + 2.0 ** -21 * size) + tiny * 2 * step
    assert ((y.double().cpu() - ref).abs() <= bound).all()


def make(shape, dtype=torch.bfloat16, seed=0):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


FREQ = {dim: dsa_amd.rotary_frequencies(dim) for dim in (2, 6, 32, 64, 128, 130, 512)}


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("tokens, heads, width, start, dim", [
    (1, 1, 64, 0, 64), (1, 128, 64, 0, 64), (3, 16, 192, 128, 64), (5, 7, 128, 0, 64), (17, 3, 128, 64, 64),
    (2, 5, 66, 1, 64), (3, 4, 6, 0, 6), (4, 2, 9, 3, 2), (2, 3, 200, 8, 130), (2, 2, 512, 0, 512), (257, 1, 64, 0, 64),
    (33, 64, 128, 0, 32), (9, 24, 96, 32, 32)])
def test_against_64_bits(tokens, heads, width, start, dim, interleaved, dtype):
    x = make((tokens, heads, width), dtype)
    positions = (torch.arange(tokens) * 977 + 5).int().cuda()
    freq = FREQ[dim].cuda()
    kept = x.clone()
    for transposed in (False, True):
        y = dsa_amd.rotary(x, positions, freq, interleaved=interleaved, start=start, transposed=transposed)
        assert y.is_contiguous() and y.dtype == dtype
        check(y, x, positions, freq, interleaved=interleaved, start=start, transposed=transposed)
        rest = [c for c in range(width) if not start <= c < start + dim]
        assert torch.equal(y[..., rest], x[..., rest])
    assert torch.equal(x, kept)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("tokens, heads, width, start, dim", [
    (2003, 40, 96, 32, 64),   # a few tokens a workgroup's run of units and a part of one
    (4999, 1, 64, 0, 64),     # many tokens a workgroup
    (61, 190, 576, 0, 512),   # several workgroups a token
    (1201, 33, 67, 3, 64)])   # nothing aligned
def test_many_units(tokens, heads, width, start, dim, interleaved, dtype):
    x = make((tokens, heads, width), dtype)
    positions = (torch.arange(tokens) * 7 + 1).cuda()
    freq = FREQ[dim].cuda()
    kw = dict(interleaved=interleaved, start=start)
    y = dsa_amd.rotary(x, positions, freq, **kw)
    check(y, x, positions, freq, **kw)
    keep = torch.ones(width, dtype=torch.bool)
    keep[start:start + dim] = False
    assert torch.equal(y[..., keep.cuda()], x[..., keep.cuda()])
    # the same by groups, in place
    if tokens % 2 == 0 or tokens == 2003:
        tokens -= tokens % 2
        z = x[:tokens].reshape(2, tokens // 2, heads, width).clone()
        dsa_amd.rotary(z, positions[:tokens].view(2, -1), freq, out=z, **kw)
        assert torch.equal(z.view(tokens, heads, width), y[:tokens])


@pytest.mark.parametrize("interleaved", [True, False])
def test_far_and_negative_positions(interleaved):
    """Positions to 2^31 - 1 in 32 bits and beyond in 64: angles of 10^9 radians."""
    freq = FREQ[64].cuda()
    far = torch.tensor([0, 1, -1, 131071, 1 << 20, -(1 << 20) - 7, (1 << 31) - 1, -(1 << 31)])
    x = make((8, 4, 64), torch.float32)
    # angle: rounded to 2^-53 of itself twice, 2^-21 radians at 2^31
    for p in (far.int().cuda(), far.cuda()):
        y = dsa_amd.rotary(x, p, freq, interleaved=interleaved)
        ref, size = exact(x, far, freq, interleaved)
        assert ((y.double().cpu() - ref).abs() <= (2.0 ** -21 + 2.0 ** -20) * size + 2.0 ** -24 * ref.abs()).all()


def test_strides_groups_and_in_place():
    freq = FREQ[64].cuda()
    big = make((3, 5, 8, 192))
    positions = torch.randint(0, 9999, (3, 5), generator=torch.Generator().manual_seed(1)).cuda()
    x = big[..., 128:]
    y = dsa_amd.rotary(x, positions, freq)
    assert y.is_contiguous()
    check(y, x, positions, freq)
    # permuted token and head dimensions, an unaligned slice, a broadcast head
    for v in (big.transpose(0, 2)[:, :, :, :64], big[..., 3:67], big[:, :, :1, :64].expand(3, 5, 8, 64)):
        p = positions if v.shape[:2] == (3, 5) else torch.arange(40).reshape(8, 5).cuda()
        check(dsa_amd.rotary(v, p, freq, interleaved=False), v, p, freq, interleaved=False)
    # in place, on the slice of a larger buffer: the rest of the buffer stays
    before = big.clone()
    whole = dsa_amd.rotary(big, positions, freq, start=128)
    r = dsa_amd.rotary(big, positions, freq, start=128, out=big)
    assert r is big and torch.equal(big, whole) and torch.equal(big[..., :128], before[..., :128])
    big.copy_(before)
    dsa_amd.rotary(x, positions, freq, out=x)
    assert torch.equal(big, whole)
    # into a cache's rows, a strided destination
    cache = torch.zeros(3, 50, 1, 128, device="cuda", dtype=torch.bfloat16)
    k = make((3, 5, 1, 128), seed=3)
    dsa_amd.rotary(k, positions, freq, interleaved=False, out=cache[:, 10:15])
    assert torch.equal(cache[:, 10:15], dsa_amd.rotary(k, positions, freq, interleaved=False))
    assert not cache[:, :10].any() and not cache[:, 15:].any()


def test_far_offsets():
    """Tokens past 2^31 elements of the input, and of the output."""
    freq, positions = FREQ[64].cuda(), torch.tensor([3, 50, 7]).cuda()
    big = torch.zeros((2 << 30) + 192, dtype=torch.bfloat16, device="cuda")
    x = big.as_strided((3, 2, 96), (1 << 30, 96, 1))
    x.copy_(make((3, 2, 96)))
    near = x.contiguous()
    want = dsa_amd.rotary(near, positions, freq, start=32)
    assert torch.equal(dsa_amd.rotary(x, positions, freq, start=32), want)
    dsa_amd.rotary(near, positions, freq, start=32, out=x)
    assert torch.equal(x, want)


def test_magnitude_and_round_trip():
    freq = FREQ[64].cuda()
    x, positions = make((6, 4, 64), torch.float32), torch.arange(6).cuda() * 1234
    y = dsa_amd.rotary(x, positions, freq, magnitude=1.5)
    check(y, x, positions, freq, magnitude=1.5)
    back = dsa_amd.rotary(y, positions, freq, transposed=True, magnitude=1 / 1.5)
    # two turns, each within 2^-21 of |x0| + |x1| <= 2 max|x|, and two roundings
    assert (back - x).abs().max() <= 2 * 2 * 2.0 ** -20 * x.abs().max()


def test_special_values_stay_in_their_pair():
    freq = FREQ[64].cuda()
    x = make((4, 2, 96), torch.float32)
    x[1, 1, 6], x[2, 0, 40], x[3, 1, 80] = float("nan"), float("inf"), float("-inf")
    y = dsa_amd.rotary(x, torch.arange(4).cuda() + 1, freq)
    assert y[1, 1, 6:8].isnan().all() and not y[2, 0, 40:42].isfinite().any() and y[3, 1, 80] == float("-inf")
    bad = torch.zeros(4, 2, 96, dtype=torch.bool)
    bad[1, 1, 6:8] = bad[2, 0, 40:42] = True
    bad[3, 1, 80] = True
    assert y.isfinite().cpu().equal(~bad)


def test_empty():
    freq = FREQ[64].cuda()
    for shape in ((0, 4, 64), (3, 0, 64), (2, 0, 4, 64)):
        y = dsa_amd.rotary(make(shape), torch.zeros(shape[:-2], dtype=torch.int32).cuda(), freq)
        assert y.shape == shape


@pytest.mark.parametrize("interleaved", [True, False])
def test_gradient(interleaved):
    """The recorded gradient is the transposed turn, and agrees with
    differences of the (linear) operator in each of a head's directions."""
    freq = FREQ[6].cuda()
    positions = torch.tensor([3, 100]).cuda()
    x = make((2, 1, 8), torch.float32).requires_grad_()
    g = make((2, 1, 8), torch.float32, seed=9)
    kw = dict(interleaved=interleaved, start=1, magnitude=0.5)
    y = dsa_amd.rotary(x, positions, freq, **kw)
    y.backward(g)
    want = dsa_amd.rotary(g, positions, freq, transposed=True, **kw)
    assert torch.equal(x.grad, want)
    base = x.detach()
    for e in range(8):
        d = torch.zeros(8, device="cuda")
        d[e] = 1.0
        diff = (dsa_amd.rotary(base + d, positions, freq, **kw) - dsa_amd.rotary(base, positions, freq, **kw)) * g
        # a difference of values up to 3 (|x| + 1), each within 2^-21 of its pair
        assert (diff.sum(-1) - want[..., e]).abs().max() <= 8 * 2.0 ** -20 * 3 * (base.abs().max() + 1) * g.abs().max()
    # the gradient of a slice, a gradient that autograd expands, and none under no_grad
    big = make((2, 4, 192)).requires_grad_()
    dsa_amd.rotary(big[..., 128:], positions, FREQ[64].cuda(), interleaved=interleaved).sum().backward()
    ones = torch.ones(2, 4, 64, device="cuda", dtype=torch.bfloat16)
    assert not big.grad[..., :128].any()
    assert torch.equal(big.grad[..., 128:],
                       dsa_amd.rotary(ones, positions, FREQ[64].cuda(), interleaved=interleaved, transposed=True))
    with torch.no_grad():
        assert not dsa_amd.rotary(big, positions, FREQ[64].cuda()).requires_grad


def test_refusals():
    f = FREQ[64].cuda()
    x, p = make((4, 2, 64)), torch.zeros(4, dtype=torch.int32).cuda()
    bad = [dict(x=x.double()), dict(x=x[..., ::2]), dict(positions=p[:3]), dict(positions=p.float()),
           dict(positions=p.cpu()), dict(positions=torch.zeros(8, dtype=torch.int32).cuda()[::2]),
           dict(frequencies=f.float()), dict(frequencies=f.cpu()), dict(frequencies=f[:0]), dict(start=1), dict(start=-1),
           dict(start=0.0), dict(magnitude=float("inf")), dict(out=torch.empty(4, 2, 64).cuda()), dict(out=x[:3]),
           dict(out=x.new_empty(1, 2, 64).expand(4, 2, 64)), dict(frequencies=FREQ[128].cuda())]
    for kw in bad:
        args = {**dict(x=x, positions=p, frequencies=f), **kw}
        with pytest.raises(ValueError):
            dsa_amd.rotary(args.pop("x"), args.pop("positions"), args.pop("frequencies"), **args)
    with pytest.raises(TypeError):
        dsa_amd.rotary(x, p, f, magnitude="1")
    shifted = make((5, 2, 64))
    with pytest.raises(ValueError, match="apart"):
        dsa_amd.rotary(shifted[:4], p, f, out=shifted[1:])
    with pytest.raises(ValueError, match="gradient"):
        dsa_amd.rotary(x.clone().requires_grad_(), p, f, out=torch.empty_like(x))


def test_other_stream_and_graph():
    """A call on another stream, and captured: replays follow the inputs."""
    f, p = FREQ[64].cuda(), torch.arange(7).cuda()
    x = make((7, 16, 192))
    want = dsa_amd.rotary(x[..., 128:], p, f)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = dsa_amd.rotary(x[..., 128:], p, f)
    side.synchronize()
    assert torch.equal(y, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = dsa_amd.rotary(x[..., 128:], p, f)
    for k in range(4):
        x.copy_(make((7, 16, 192), seed=k))
        p.copy_(torch.arange(7) * (k + 1))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, dsa_amd.rotary(x[..., 128:], p, f))


def test_captured_gradient():
    """Forward and backward in one captured graph, replayed with new inputs between eager calls."""
    freq, positions = FREQ[64].cuda(), torch.arange(9).cuda() * 31
    x, w = make((9, 3, 96), torch.float32).requires_grad_(), make((9, 3, 96), torch.float32, seed=1)

    def step(x):
        y = dsa_amd.rotary(x, positions, freq, start=16, magnitude=1.5)
        return y, torch.autograd.grad(y, x, w)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(x)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, dx = step(x)
    for k in range(4):
        with torch.no_grad():
            x.copy_(make((9, 3, 96), torch.float32, seed=2 + k))
            w.copy_(make((9, 3, 96), torch.float32, seed=20 + k))
            positions.add_(1000)
        graph.replay()
        other = step(x.detach().clone().requires_grad_())
        assert torch.equal(y, other[0]) and torch.equal(dx, other[1])
        torch.cuda.synchronize()
