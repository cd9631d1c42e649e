"""Norms of rows whose squares leave the range of 32 bits, and the errors of ordinary
ones, against plain forms in 64 bits.

Tolerances.  A thread adds up 8 squares (16 in rows above 8192), a wave in 6 steps, a
row over 16 waves at most: 38 roundings of 2^-24, all terms positive.  eps, the mean (two:
a unit in the last place is allowed for quotients and the root) and their sum are four
more, and the root halves them: 21.  The root, its reciprocal and two products are six
behind it: fewer than 32 in all, SUM = 2^-19, and half a step of the output's type.  Where
a value is below the type's range its first product is off by 2^-150, times the weight.

The gradient's mean has as many roundings, 38, of sum |b u| / n, u = h / rms 26, b 1, the
quotient 2: 67; u times it 94, the difference, its product with 1 / rms and the addition
28 more: fewer than 128.  The weight's gradient: u 26, the rows of a team one after the
other, a group's share of the teams' sums (every 32nd), and 32 groups.
"""
import math

import pytest
import torch

import dsa_amd
from test_gpu_norm import check_codes, gradients, half_step, least, make, normed

pytestmark = pytest.mark.gpu

BF, HALF, FULL = torch.bfloat16, torch.float16, torch.float32
SUM = 32 * 2.0 ** -24


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm GPU")
    torch.cuda.init()


def check_norm(x, weight, residual, eps):
    out = dsa_amd.rms_norm(x, weight, residual, eps=eps)
    y, h = out if residual is not None else (out, x)
    want = normed(h, weight, eps)
    bound = want.abs() * (half_step(x.dtype) + SUM) * (1 + 2.0 ** -8) + least(x.dtype)
    bound += 2.0 ** -149 * (1 + weight.double().abs())
    assert ((y.double() - want).abs() <= bound).all()
    return y


WIDTHS = [1, 7, 64, 100, 512, 520, 1000, 1536, 2049, 4096, 7168, 8192, 8200, 16384]


@pytest.mark.parametrize("dtype", [BF, HALF, FULL])
@pytest.mark.parametrize("dim", WIDTHS)
def test_ordinary_rows(dim, dtype):
    x, w, r = make((67, dim), dtype), make(dim, dtype, 1), make((67, dim), dtype, 2)
    check_norm(x, w, None, 1e-6)
    check_norm(x, w.float(), r, 0.5)


@pytest.mark.parametrize("dim", WIDTHS)
@pytest.mark.parametrize("power, dtype", [(-145, FULL)] + [(power, dtype) for dtype in (BF, FULL) for power in
                                                            (-127, -126, -100, -75, -63, -49, -45, 55, 62, 64, 100, 120)])
def test_rows_of_any_size(power, dtype, dim):
    """Values of 2^power, eps 0 or as large as their squares, ordinary rows between them."""
    size = 2.0 ** power
    x = make((6, dim), FULL, 3).abs() + 0.25
    x[::2] *= -1.0
    x[1::2] = (x[1::2].double() * size).clamp(-3e38, 3e38).float()
    x = x.to(dtype)
    w, r = make(dim, dtype, 1), torch.zeros(6, dim, dtype=dtype, device="cuda")
    for eps in (0.0, min(max(size * size, 1e-37), 1e38), 1e-6):
        check_norm(x, w, None, eps)
        check_norm(x, w, r, eps)


@pytest.mark.parametrize("dim", [1, 300, 1536, 16384])
def test_one_value_in_a_row(dim):
    """The rest of it zeros: its place's weight times the root of dim."""
    for value in (1e-45, 1e-38, 1e-30, 1e19, 2e19, 3e38):
        for at in {0, dim // 2, dim - 1}:
            x = torch.zeros(3, dim, device="cuda")
            x[1, at] = value
            y = check_norm(x[1:2], make(dim, FULL, 1), None, 0.0)
            assert torch.count_nonzero(y) <= 1
            check_norm(x, make(dim, FULL, 1), None, 1e-30)


@pytest.mark.parametrize("dim", [16, 144, 1536, 8208])
@pytest.mark.parametrize("pow2", [True, False])
@pytest.mark.parametrize("value", [1e-44, 1e-38, 1e-23, 1e22, 1e38])
def test_codes_of_rows_of_any_size(value, pow2, dim):
    """The last block is short, and some values are zero."""
    x, w = (make((5, dim), FULL, 4).double().clamp(-3, 3) * value).float(), make(dim, BF, 1).float()
    x[:, ::5] = 0.0
    got = dsa_amd.rms_norm_fp8(x, w, eps=0.0, pow2_scales=pow2)
    check_codes(got, normed(x, w, 0.0), pow2)
    got = dsa_amd.rms_norm_fp8(x, w, torch.zeros_like(x), eps=0.0, pow2_scales=pow2)
    check_codes(got, normed(x, w, 0.0), pow2)


def test_special_rows_among_them():
    """Rows that no power of two helps, one after the other in a team's turn."""
    for dim in (512, 3000):
        x, w = make((9000, dim), FULL), make(dim, FULL, 1)
        clean = dsa_amd.rms_norm(x, w, eps=0.0)
        x[::4], x[1::4, 3], x[2::4, 5] = 0.0, math.inf, math.nan
        y = dsa_amd.rms_norm(x, w, eps=0.0)
        assert y[::4].isnan().all() and y[2::4].isnan().all() and torch.equal(y[3::4], clean[3::4])
        assert y[1::4, 3].isnan().all() and not y[1::4, :3].any() and not y[1::4, 4:].any()


def check_gradients(x, weight, residual, eps):
    leaves = [t.detach().requires_grad_() for t in (x, weight, residual) if t is not None]
    out = dsa_amd.rms_norm(leaves[0], leaves[1], *leaves[2:], eps=eps)
    out = out if isinstance(out, tuple) else (out,)
    given = [make(x.shape, x.dtype, 7 + i) for i in range(len(out))]
    got = torch.autograd.grad(out, leaves, given)
    h = out[1].detach() if residual is not None else x
    dh, size, dw, wsize = gradients(h, weight, eps, given[0], given[1] if residual is not None else None)
    rows, dim = x.shape
    bound = half_step(x.dtype) * dh.abs() * (1 + 2.0 ** -8) + 128 * 2.0 ** -24 * size + least(x.dtype)
    assert ((got[0].double() - dh).abs() <= bound).all()
    teams = 4 if dim <= 512 else 1
    teams *= min(512, -(-rows // teams))
    deep = 26 + -(-rows // teams) + -(-teams // 32) + 32
    bound = half_step(weight.dtype) * dw.abs() * (1 + 2.0 ** -8) + deep * 2.0 ** -24 * wsize + least(weight.dtype)
    assert ((got[1].double() - dw).abs() <= bound).all()


@pytest.mark.parametrize("dtype", [BF, HALF, FULL])
@pytest.mark.parametrize("rows, dim", [(1, 7), (5, 64), (67, 512), (5, 1000), (515, 4096), (3, 8200), (4100, 512), (1030, 7168)])
def test_gradients(rows, dim, dtype):
    x, w, r = make((rows, dim), dtype), make(dim, dtype, 1), make((rows, dim), dtype, 2)
    check_gradients(x, w, None, 1e-6)
    check_gradients(x, w.float(), r, 0.1)


@pytest.mark.parametrize("dim", [7, 512, 1536, 16384])
@pytest.mark.parametrize("power", [-100, -70, 62, 100])
def test_gradients_of_rows_of_any_size(power, dim):
    """Of finite size: 1 / rms below 2^101."""
    x = (make((5, dim), FULL, 3).abs() + 0.25) * 2.0 ** power
    check_gradients(x, make(dim, FULL, 1), None, 0.0)
    check_gradients(x, make(dim, FULL, 1), torch.zeros_like(x), 0.0)
