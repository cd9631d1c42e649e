"""Norms, their gradients and 8-bit codes against plain forms in 64 bits.

Tolerances.  A row's sum of squares is at most 64 products deep in a thread, 6
additions in a wave and 16 over waves, all positive: 86 roundings of 2^-24, halved by
the root; with the mean, eps, root, reciprocal and two products fewer than 50 in all,
64 x 2^-24 = 2^-18 of a value, and half a step of the output's type beside it.  The
gradient's mean has as many roundings, of sum |b u| / n.
"""
import math

import pytest
import torch

import dsa_amd

pytestmark = pytest.mark.gpu

BF, HALF, FULL = torch.bfloat16, torch.float16, torch.float32
SUM = 64 * 2.0 ** -24


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm GPU")
    torch.cuda.init()


def make(shape, dtype=BF, seed=0, gain=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * gain).to(dtype).cuda()


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def least(dtype):
    return torch.finfo(dtype).tiny * torch.finfo(dtype).eps


def normed(h, weight, eps):
    h = h.double()
    return h / (h.square().mean(-1, keepdim=True) + eps).sqrt() * weight.double()


def check_norm(x, weight, residual, eps=1e-6):
    out = dsa_amd.rms_norm(x, weight, residual, eps=eps)
    if residual is None:
        y, h = out, x
    else:
        y, h = out
        assert h.dtype == x.dtype and h.is_contiguous() and torch.equal(h, x + residual)
    assert y.dtype == x.dtype and y.shape == x.shape and y.is_contiguous() and not y.requires_grad
    want = normed(h, weight, eps)
    bound = want.abs() * (half_step(x.dtype) + SUM) * (1 + 2.0 ** -8) + least(x.dtype)
    assert ((y.double() - want).abs() <= bound).all()


@pytest.mark.parametrize("dtype", [BF, HALF, FULL])
@pytest.mark.parametrize("rows, dim", [(1, 1), (3, 7), (5, 8), (9, 64), (4, 100), (65, 512), (3, 513), (7, 520), (6, 1000),
                                       (5, 1024), (3, 1536), (2, 2048), (2, 2049), (3, 4096), (1, 7168), (3, 8192), (2, 8200),
                                       (2, 16383), (3, 16384), (700, 1536), (530, 4100), (515, 7168), (520, 16384)])
def test_against_64_bits(rows, dim, dtype):
    weight = make(dim, dtype, 1)
    check_norm(make((rows, dim), dtype), weight, None)
    check_norm(make((rows, dim), dtype), weight, make((rows, dim), dtype, 2))
    check_norm(make((rows, dim), dtype, 3, 100.0), weight.float(), make((rows, dim), dtype, 4), eps=0.5)


@pytest.mark.parametrize("rows, dim", [(20011, 512), (5003, 1536), (4999, 4096)])
def test_many_rows(rows, dim):
    """More rows than workgroups."""
    check_norm(make((rows, dim)), make(dim, seed=1), make((rows, dim), seed=2))


def test_strides_and_alignment():
    wide = make((6, 5, 600))
    weight = make(512, seed=1)
    for x in (wide[..., :512], wide[..., 8:520], wide[..., 1:513], wide[::2, :, :512][:, 0], wide[:1, :, 3:515],
              wide.transpose(0, 1)[:, 0, :512], make((1, 1, 512)).expand(1, 4, 512), make((3, 512))[1]):
        check_norm(x, weight, None)
        check_norm(x, weight, make(x.shape, seed=5))
        check_norm(make(x.shape, seed=6), weight, x)
    check_norm(wide[0, 0, :512], make(520, seed=2)[3:515], None)
    for bad in (wide[:, ::2].transpose(0, 1)[..., :512], wide[..., ::2]):
        with pytest.raises(ValueError, match="evenly spaced"):
            dsa_amd.rms_norm(bad, make(bad.shape[-1]))


def test_far_offsets():
    """Rows more than 2^31 elements apart."""
    apart = (1 << 31) + 64
    store = torch.empty(apart + 1024, dtype=BF, device="cuda")
    x = store.as_strided((2, 1024), (apart, 1))
    x.copy_(make((2, 1024)))
    check_norm(x, make(1024, seed=1), None)
    codes, scales = dsa_amd.quantize_fp8(x)
    other = dsa_amd.quantize_fp8(x.contiguous())
    assert torch.equal(codes.view(torch.uint8), other[0].view(torch.uint8)) and torch.equal(scales, other[1])


def test_special_rows():
    """Zeros, infinities and NaN stay in their row, and go by the formula."""
    x = make((5, 640), FULL)
    clean = dsa_amd.rms_norm(x, make(640, FULL, 1))
    x[0], x[1, 3], x[2, 639] = 0.0, math.inf, math.nan
    y = dsa_amd.rms_norm(x, make(640, FULL, 1))
    assert not y[0].any() and torch.equal(y[3:], clean[3:])
    assert y[1, 3].isnan() and not y[1, :3].any() and y[2].isnan().all()
    assert dsa_amd.rms_norm(x[:1], make(640, FULL, 1), eps=0.0).isnan().all()


def test_empty():
    for shape in ((0, 512), (3, 0, 512)):
        x = make(shape)
        y, h = dsa_amd.rms_norm(x, make(512), x)
        assert y.shape == h.shape == shape
        codes, scales, h = dsa_amd.rms_norm_fp8(x, make(512), x)
        assert codes.shape == shape and scales.shape == (*shape[:-1], 4) and h.shape == shape
    x, w = make((0, 512)).requires_grad_(), make(512).requires_grad_()
    gx, gw = torch.autograd.grad(dsa_amd.rms_norm(x, w).sum(), (x, w))
    assert gx.shape == (0, 512) and not gw.any()


# ------------------------------------------------------------ gradients

def gradients(h, weight, eps, gy, gh):
    """By the formula, in 64 bits, and what its terms add up to."""
    h, w, gy = h.double(), weight.double(), gy.double()
    inverse = 1 / (h.square().mean(-1, keepdim=True) + eps).sqrt()
    u, b = h * inverse, gy * w
    dh = (b - u * (b * u).mean(-1, keepdim=True)) * inverse + (0 if gh is None else gh.double())
    size = (b.abs() + u.abs() * (b * u).abs().mean(-1, keepdim=True)) * inverse + (0 if gh is None else gh.double().abs())
    flat = (gy * u).flatten(0, -2)
    return dh, size, flat.sum(0), flat.abs().sum(0)


def check_gradients(x, weight, residual, seed=0, eps=1e-6):
    leaves = [t.detach().requires_grad_() for t in (x, weight, residual) if t is not None]
    out = dsa_amd.rms_norm(leaves[0], leaves[1], leaves[2] if residual is not None else None, eps=eps)
    out = out if isinstance(out, tuple) else (out,)
    given = [make(x.shape, x.dtype, seed + 7 + i) for i in range(len(out))]
    got = torch.autograd.grad(out, leaves, given)
    h = out[1].detach() if residual is not None else x
    dh, size, dw, wsize = gradients(h, weight, eps, given[0], given[1] if residual is not None else None)
    rows = x.numel() // x.shape[-1]
    # b has 51 roundings, u 50, their mean 86 more; the weight's sum is at most rows / 512 + 1 rows in a team,
    # 128 teams a group and 16 groups deep
    bound = half_step(x.dtype) * dh.abs() * (1 + 2.0 ** -8) + 256 * 2.0 ** -24 * size + least(x.dtype)
    assert got[0].shape == x.shape and ((got[0].double() - dh).abs() <= bound).all()
    deep = 51 + rows / 512 + 1 + 128 + 16
    bound = half_step(weight.dtype) * dw.abs() * (1 + 2.0 ** -8) + deep * 2.0 ** -24 * wsize + least(weight.dtype)
    assert got[1].dtype == weight.dtype and ((got[1].double() - dw).abs() <= bound).all()
    if residual is not None:
        assert torch.equal(got[2], got[0])
    return got


@pytest.mark.parametrize("dtype", [BF, HALF, FULL])
@pytest.mark.parametrize("rows, dim", [(1, 1), (3, 7), (5, 64), (9, 100), (65, 512), (7, 520), (5, 1000), (6, 1024), (3, 1536),
                                       (2, 2049), (3, 4096), (515, 4096), (2, 7168), (2, 8200), (3, 16384), (2100, 512),
                                       (2500, 300)])
def test_gradients(rows, dim, dtype):
    x, residual = make((rows, dim), dtype), make((rows, dim), dtype, 2)
    check_gradients(x, make(dim, dtype, 1), None)
    check_gradients(x, make(dim, dtype, 1), residual)
    check_gradients(x, make(dim, FULL, 1), residual, eps=0.1)


def test_gradients_are_differences_of_the_formula():
    """Central differences of sum(gy y + gh h) in 64 bits, in a few directions:
    third derivatives of a sum of 96 such terms stay below 2^10, a step of 2^-12 is
    off by 2^-24 x 2^10 / 6 and its roundings by 2^12 x 2^-50."""
    x, w, residual = make((4, 96), FULL), make(96, FULL, 1), make((4, 96), FULL, 2)
    got = check_gradients(x, w, residual)
    gy, gh = make((4, 96), FULL, 7).double(), make((4, 96), FULL, 8).double()
    h = (x + residual).double()

    def loss(h, w):
        return (gy * normed(h, w, 1e-6) + gh * h).sum().item()

    for seed in range(5):
        dh, dw = make((4, 96), FULL, 30 + seed).double(), make(96, FULL, 60 + seed).double()
        step = 2.0 ** -12
        rise = (loss(h + step * dh, w.double() + step * dw) - loss(h - step * dh, w.double() - step * dw)) / (2 * step)
        along = (got[0].double() * dh).sum().item() + (got[1].double() * dw).sum().item()
        assert abs(rise - along) <= 2.0 ** -10


def test_gradients_of_parts():
    """Of some of the inputs, of one output, of strided, shared and expanded inputs, twice added."""
    wide, w = make((6, 600)), make(512, seed=1)
    check_gradients(wide[:, 3:515], w, None)
    check_gradients(wide[:, :512], w, make((6, 512), seed=2))
    x, r = make((6, 512), FULL), make((6, 512), FULL, 2)
    w = make(512, FULL, 1)
    full = check_gradients(x, w, r)
    gy, gh = make((6, 512), FULL, 7), make((6, 512), FULL, 8)
    leaf = x.clone().requires_grad_()
    y, h = dsa_amd.rms_norm(leaf, w, r)
    assert torch.equal(torch.autograd.grad((y, h), leaf, (gy, gh))[0], full[0])
    leaf = w.clone().requires_grad_()
    y, h = dsa_amd.rms_norm(x, leaf, r)
    assert torch.equal(torch.autograd.grad(y, leaf, gy)[0], full[1])
    leaf = r.clone().requires_grad_()
    only, = torch.autograd.grad(dsa_amd.rms_norm(x, w, leaf)[1], leaf, gh)
    assert torch.equal(only, gh)
    row = x[:1].clone().requires_grad_()
    got, = torch.autograd.grad(dsa_amd.rms_norm(row.expand(6, 512), w, r)[0], row, gy)
    leaf = x[:1].expand(6, 512).contiguous().requires_grad_()
    each, = torch.autograd.grad(dsa_amd.rms_norm(leaf, w, r)[0], leaf, gy)
    assert torch.allclose(got, each.sum(0, keepdim=True), rtol=1e-5, atol=1e-5)
    same = x.clone().requires_grad_()  # both summands
    got, = torch.autograd.grad(dsa_amd.rms_norm(same, w, same)[0], same, gy)
    leaf = x.clone().requires_grad_()
    once, = torch.autograd.grad(dsa_amd.rms_norm(leaf, w, x)[0], leaf, gy)
    assert torch.equal(got, once + once)
    same.grad = None
    for _ in range(2):
        y, h = dsa_amd.rms_norm(same, w, r)
        (y * gy + h * gh).sum().backward()
    assert torch.allclose(same.grad, 2 * full[0], rtol=1e-6, atol=1e-6)


def test_a_saved_input_that_was_written_is_noticed():
    x, w = make((4, 512)).requires_grad_(), make(512)
    y = dsa_amd.rms_norm(x, w)
    with torch.no_grad():
        x.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_no_second_order_and_no_tangent():
    x, w = make((2, 64), FULL).requires_grad_(), make(64, FULL, 1)
    g, = torch.autograd.grad(dsa_amd.rms_norm(x, w).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.sum().backward()
    import torch.autograd.forward_ad as fwd
    with fwd.dual_level():
        with pytest.raises(ValueError, match="forward-mode"):
            dsa_amd.rms_norm(fwd.make_dual(x.detach(), torch.ones_like(x)), w)
        with pytest.raises(ValueError, match="tangent"):
            dsa_amd.rms_norm_fp8(fwd.make_dual(x.detach(), torch.ones_like(x)), w)


# ------------------------------------------------------------ 8-bit codes

def check_codes(got, v, pow2):
    """Codes and scales against values ``v`` in 64 bits: a code is half a step, 2^-4, from
    its value, or half the least one's, 2^-10; the value itself has errors of SUM."""
    codes, scales = got[:2]
    dim = v.shape[-1]
    blocks = -(-dim // 128)
    assert codes.dtype == torch.float8_e4m3fn and codes.shape == v.shape and scales.shape == (*v.shape[:-1], blocks)
    wide = torch.nn.functional.pad(v, (0, blocks * 128 - dim)).unflatten(-1, (blocks, 128))
    top = wide.abs().amax(-1) / 448.0
    scales = scales.double()
    if pow2:
        assert (torch.frexp(scales)[0] == 0.5).all()
        exact = torch.where(top > 0, torch.exp2(torch.ceil(torch.log2(top))), 1.0)
        near = (torch.frexp(top)[0] - 0.5).abs() < 2.0 ** -17  # the quotient is a power of two, or all but one
        near |= (torch.frexp(top)[0] - 1.0).abs() < 2.0 ** -17
        assert ((scales == exact) | (near & ((scales == 2 * exact) | (2 * scales == exact)))).all()
    else:
        exact = torch.where(top > 0, top, 1.0)
        assert ((scales - exact).abs() <= exact * (SUM + 2.0 ** -22)).all()
    each = scales.repeat_interleave(128, -1)[..., :dim]
    value = v / each
    bound = value.abs() * (2.0 ** -4 + 2.0 ** -16) + 2.0 ** -10 * (1 + 2.0 ** -16)
    assert ((codes.double() - value).abs() <= bound).all()


@pytest.mark.parametrize("dtype", [BF, HALF, FULL])
@pytest.mark.parametrize("pow2", [True, False])
@pytest.mark.parametrize("rows, dim", [(1, 16), (5, 112), (4, 128), (3, 144), (65, 512), (3, 528), (6, 1008), (2, 2064),
                                       (3, 4096), (2, 7168), (3, 16384), (2, 8208), (700, 1536), (520, 7168), (9000, 128)])
def test_codes(rows, dim, pow2, dtype):
    x, weight, residual = make((rows, dim), dtype), make(dim, dtype, 1), make((rows, dim), dtype, 2)
    got = dsa_amd.rms_norm_fp8(x, weight, residual, pow2_scales=pow2)
    assert torch.equal(got[2], x + residual)
    check_codes(got, normed(got[2], weight, 1e-6), pow2)
    check_codes(dsa_amd.rms_norm_fp8(x, weight.float(), eps=0.1, pow2_scales=pow2), normed(x, weight, 0.1), pow2)
    check_codes(dsa_amd.quantize_fp8(x, pow2_scales=pow2), x.double(), pow2)


def test_codes_are_the_cache_rows():
    """The same codes and scales as an fp8 cache row's."""
    x = make((300, 512), gain=3.0)
    rows = dsa_amd.quantize_kv_fp8(x, x[:, :64])
    codes, scales = dsa_amd.quantize_fp8(x)
    assert torch.equal(codes.view(torch.uint8), rows[:, :512]) and torch.equal(scales, rows[:, 512:528].contiguous().view(FULL))


def test_codes_of_strided_and_unaligned_rows():
    wide = make((6, 5, 600))
    for x in (wide[..., :512], wide[..., 8:520], wide[..., 1:513], wide[:1, :, 3:515], make((3, 512))[1]):
        for pow2 in (True, False):
            got, want = dsa_amd.quantize_fp8(x, pow2_scales=pow2), dsa_amd.quantize_fp8(x.contiguous(), pow2_scales=pow2)
            assert torch.equal(got[0].view(torch.uint8), want[0].view(torch.uint8)) and torch.equal(got[1], want[1])


def test_special_codes():
    """Zeros, the largest and least numbers, infinities and NaN: each in its own block."""
    for pow2 in (True, False):
        x = make((1, 7 * 128), FULL)
        want = dsa_amd.quantize_fp8(x, pow2_scales=pow2)
        x[0, 128:256] = 0.0
        x[0, 300] = math.inf
        x[0, 400] = math.nan
        x[0, 512:640] *= 1e-42
        x[0, 700] = 3e38
        codes, scales = dsa_amd.quantize_fp8(x, pow2_scales=pow2)
        c = codes.float()
        assert torch.equal(c[0, :128], want[0].float()[0, :128]) and torch.equal(c[0, 768:], want[0].float()[0, 768:])
        assert scales[0, 0] == want[1][0, 0] and scales[0, 6] == want[1][0, 6]
        assert not c[0, 128:256].any() and scales[0, 1] == 1.0
        assert scales[0, 2] == math.inf and c[0, 300].isnan() and c[0, 256:384].nan_to_num(0.0).abs().max() == 0.0
        assert c[0, 400].isnan() and c[0, 384:512].isnan().sum() == 1 and scales[0, 3] == 1.0
        back = c[0, 512:640].double() * scales[0, 4].double()
        # a scale of so few steps is off by half of one, 2^-150, and the largest code stands for 448 of them
        most = x[0, 512:640].double().abs().max() * 2.0 ** -4 + 2.0 ** -148 + 448 * 2.0 ** -150
        assert ((back - x[0, 512:640].double()).abs() <= most).all()
        assert c[0, 640:768].isfinite().all()
        assert (c[0, 700].double() * scales[0, 5].double()).item() == pytest.approx(3e38, rel=2.0 ** -4)


# ------------------------------------------------------------ streams, graphs, refusals

def test_repeats_streams_and_graphs():
    x, w, r = make((77, 1536)), make(1536, seed=1), make((77, 1536), seed=2)
    want = [t.clone() for t in dsa_amd.rms_norm(x, w, r)]
    codes = dsa_amd.rms_norm_fp8(x, w, r)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = dsa_amd.rms_norm(x, w, r)
    side.synchronize()
    for a, b in zip(want, other):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, h = dsa_amd.rms_norm(x, w, r)
        codes = dsa_amd.rms_norm_fp8(h, w)
    for k in range(4):
        x.copy_(make((77, 1536), seed=10 + k))
        graph.replay()
        again = dsa_amd.rms_norm(x, w, r)
        assert torch.equal(y, again[0]) and torch.equal(h, again[1])
        for a, b in zip(codes, dsa_amd.rms_norm_fp8(h, w)):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
        torch.cuda.synchronize()


def test_captured_gradients():
    x, w, r = (make(s, FULL, i).requires_grad_() for i, s in enumerate([(600, 520), (520,), (600, 520)]))
    gy, gh = make((600, 520), FULL, 7), make((600, 520), FULL, 8)

    def step(x, w, r):
        out = dsa_amd.rms_norm(x, w, r)
        return (*out, *torch.autograd.grad(out, (x, w, r), (gy, gh)))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(x, w, r)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(x, w, r)
    for k in range(4):
        with torch.no_grad():
            x.copy_(make((600, 520), FULL, 20 + k))
            w.copy_(make(520, FULL, 30 + k))
            gy.copy_(make((600, 520), FULL, 40 + k))
        graph.replay()
        want = step(*(t.detach().clone().requires_grad_() for t in (x, w, r)))
        for a, b in zip(got, want):
            assert torch.equal(a, b)
        torch.cuda.synchronize()


def test_a_capture_beside_a_living_graph_is_refused():
    """The leaves' sums of an eager graph on the default stream cannot be captured: the call says so, and nothing
    is lost.  Without that graph, or without gradients, it is captured."""
    x, w = make((40, 512), FULL).requires_grad_(), make(512, FULL, 1).requires_grad_()
    kept = dsa_amd.rms_norm(x, w)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for call in (lambda: dsa_amd.rms_norm(x, w), lambda: dsa_amd.rms_norm(x.detach(), w),
                     lambda: dsa_amd.rms_norm(x, w, eps=0)):  # eps as an int: checked in Python
            with pytest.raises(ValueError, match="captured"):
                call()
        with torch.no_grad():
            plain = dsa_amd.rms_norm(x, w)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(plain, kept)
    del kept
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        (got,) = torch.autograd.grad(dsa_amd.rms_norm(x, w), w, x.detach())
    graph.replay()
    torch.cuda.synchronize()
    (want,) = torch.autograd.grad(dsa_amd.rms_norm(x, w), w, x.detach())
    assert torch.equal(got, want)


def test_one_tensor_twice():
    """x as its own residual: both summands' gradients arrive."""
    x, w, g = make((33, 520), FULL).requires_grad_(), make(520, FULL, 1), make((33, 520), FULL, 2)
    y, h = dsa_amd.rms_norm(x, w, x)
    assert torch.equal(h, 2 * x)
    (got,) = torch.autograd.grad((y, h), x, (g, g))
    a, b = x.detach().clone().requires_grad_(), x.detach().clone().requires_grad_()
    one, other = torch.autograd.grad(dsa_amd.rms_norm(a, w, b), (a, b), (g, g))
    assert torch.equal(got, one + other)


def test_views_of_the_other_sign():
    """Views that keep their sign apart from their memory are taken by their values."""
    x, w, r, g = make((9, 256), FULL), make(256, FULL, 1), make((9, 256), FULL, 2), make((9, 256), FULL, 3)
    other = torch._neg_view
    assert other(x).is_neg()
    want = dsa_amd.rms_norm(-x, -w, -r)
    for a, b in zip(want, dsa_amd.rms_norm(other(x), other(w), other(r))):
        assert torch.equal(a, b)
    for a, b in zip(dsa_amd.rms_norm_fp8(-x, w, -r) + dsa_amd.quantize_fp8(-x),
                    dsa_amd.rms_norm_fp8(other(x), w, other(r)) + dsa_amd.quantize_fp8(other(x))):
        assert torch.equal(a.float(), b.float())
    for eps in (1e-6, 0):  # eps as an int: the Python path's backward
        x1, r1 = x.clone().requires_grad_(), r.clone().requires_grad_()
        want = torch.autograd.grad(dsa_amd.rms_norm(x1, w, r1, eps=eps), (x1, r1), (-g, -g))
        got = torch.autograd.grad(dsa_amd.rms_norm(x1, w, r1, eps=eps), (x1, r1), (other(g), other(g)))
        for a, b in zip(want, got):
            assert torch.equal(a, b)


def test_refusals():
    x, w = make((4, 512)), make(512)
    bad = [dict(x=x.double()), dict(x=x.cpu()), dict(x=x[:, ::2], weight=w[:256]), dict(x=None), dict(weight=None),
           dict(weight=w[:511]), dict(weight=w.half()), dict(weight=w.cpu()), dict(weight=w[None]),
           dict(weight=make(1024)[::2]), dict(residual=x[:3]), dict(residual=x.float()), dict(residual=x.cpu()),
           dict(residual=1), dict(eps=-1.0), dict(eps=math.nan), dict(eps=math.inf), dict(x=make((2, 16400)), weight=make(16400)),
           dict(x=make((2, 0)), weight=make(0))]
    for call in (dsa_amd.rms_norm, dsa_amd.rms_norm_fp8):
        for kw in bad:
            with pytest.raises(ValueError):
                call(**{**dict(x=x, weight=w), **kw})
        for eps in ("1", True, None):
            with pytest.raises(TypeError):
                call(x, w, eps=eps)
    for kw in (dict(x=make((4, 520))), dict(x=x.clone().requires_grad_()), dict(x=x[:, :8])):
        with pytest.raises(ValueError):
            dsa_amd.quantize_fp8(**kw)
    with pytest.raises(ValueError, match="gradient"):
        dsa_amd.rms_norm_fp8(x, w.clone().requires_grad_())
    with torch.no_grad():
        dsa_amd.rms_norm_fp8(x, w.clone().requires_grad_())
        assert not dsa_amd.rms_norm(x, w.clone().requires_grad_()).requires_grad
