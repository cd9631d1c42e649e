"""What a NaN or an infinity does to the 8-bit codes of its block: as the docstrings and
include/dsa_mi355x_layer.h say, value by value."""
import math

import pytest
import torch

import dsa_amd

pytestmark = pytest.mark.gpu

BF, FULL = torch.bfloat16, torch.float32


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm GPU")
    torch.cuda.init()


def rows(dtype, dim):
    g = torch.Generator().manual_seed(dim)
    return torch.randn(4, dim, generator=g).to(dtype).cuda()


@pytest.mark.parametrize("pow2", [True, False])
@pytest.mark.parametrize("dtype", [BF, FULL])
@pytest.mark.parametrize("dim, at", [(16, 0), (128, 0), (400, 384), (2048, 512), (7168, 1152)])
def test_a_nan_makes_its_blocks_scale_1(dim, at, dtype, pow2):
    """Its block's other values are coded as they are: past 448 as 448, below 2^-10 as 0."""
    x = rows(dtype, dim)
    clean = dsa_amd.quantize_fp8(x, pow2_scales=pow2)
    given = [math.nan, 1e4, -1e4, 1e-4, 2.0 ** -10, 1.5 * 2.0 ** -10, 3.0, -2.5, 448.0, 460.0, math.inf, -math.inf, 0.0]
    coded = [math.nan, 448.0, -448.0, 0.0, 0.0, 2.0 ** -9, 3.0, -2.5, 448.0, 448.0, 448.0, -448.0, 0.0]
    x[1, at:at + 13] = torch.tensor(given, device="cuda").to(dtype)
    codes, scales = dsa_amd.quantize_fp8(x, pow2_scales=pow2)
    assert torch.equal(codes[1, at:at + 13].float().nan_to_num(-1.0), torch.tensor(coded, device="cuda").nan_to_num(-1.0))
    assert scales[1, at // 128] == 1.0
    rest, other = torch.ones(4, dim, dtype=torch.bool, device="cuda"), torch.ones(scales.shape, dtype=torch.bool, device="cuda")
    rest[1, at // 128 * 128:at // 128 * 128 + 128] = False
    other[1, at // 128] = False
    assert torch.equal(codes.float()[rest], clean[0].float()[rest]) and torch.equal(scales[other], clean[1][other])


@pytest.mark.parametrize("pow2", [True, False])
@pytest.mark.parametrize("dtype", [BF, FULL])
@pytest.mark.parametrize("value", [math.inf, -math.inf])
def test_an_infinity_makes_its_blocks_scale_infinite(value, dtype, pow2):
    """Its own code is NaN, the others' 0."""
    x = rows(dtype, 384)
    x[1, 200], x[2, 140:150] = value, value
    codes, scales = dsa_amd.quantize_fp8(x, pow2_scales=pow2)
    want = torch.zeros(4, 384, dtype=torch.bool, device="cuda")
    want[1, 200], want[2, 140:150] = True, True
    assert torch.equal(codes.float().isnan(), want)
    assert torch.equal(scales == math.inf, want.unflatten(1, (3, 128)).any(-1))
    assert not codes.float()[want.unflatten(1, (3, 128)).any(-1).repeat_interleave(128, 1) & ~want].any()


@pytest.mark.parametrize("pow2", [True, False])
def test_a_norms_special_rows(pow2):
    """A row with a NaN is NaN throughout; one with an infinity is 0 but there, where it is NaN."""
    x, w = rows(BF, 400), torch.ones(400, dtype=BF, device="cuda")
    clean = dsa_amd.rms_norm_fp8(x, w, pow2_scales=pow2)
    x[1, 7], x[2, 390] = math.nan, math.inf
    codes, scales = dsa_amd.rms_norm_fp8(x, w, pow2_scales=pow2)
    codes = codes.float()
    assert codes[1].isnan().all() and codes[2, 390].isnan() and not codes[2, :390].any() and not codes[2, 391:].any()
    assert (scales[1:3] == 1.0).all()
    assert torch.equal(codes[[0, 3]], clean[0].float()[[0, 3]]) and torch.equal(scales[[0, 3]], clean[1][[0, 3]])
