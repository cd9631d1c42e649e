"""matmul_fp8 records no derivative, and says so where one is asked for."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

import dsa_amd
from dsa_amd import api

pytestmark = pytest.mark.gpu

NAMES = ("a", "a_scales", "b", "b_scales")


@pytest.fixture
def inputs():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm GPU")
    g = torch.Generator().manual_seed(0)
    e4m3 = torch.float8_e4m3fn
    return dict(a=torch.randn(5, 256, generator=g).to(e4m3).cuda(), a_scales=torch.rand(5, 2, generator=g).cuda(),
                b=torch.randn(200, 256, generator=g).to(e4m3).cuda(), b_scales=torch.rand(2, 2, generator=g).cuda())


@pytest.mark.parametrize("name", NAMES)
def test_a_gradient_is_refused(inputs, name):
    want = dsa_amd.matmul_fp8(**inputs)
    asked = {**inputs, name: inputs[name].clone().requires_grad_()}
    assert api._fast_layer().matmul_fp8(*asked.values(), torch.bfloat16) is None
    with pytest.raises(ValueError, match="no gradient"):
        dsa_amd.matmul_fp8(**asked)
    for off in (torch.no_grad, torch.inference_mode):
        with off():
            got = dsa_amd.matmul_fp8(**asked)
        assert torch.equal(got, want) and not got.requires_grad
    assert torch.equal(dsa_amd.matmul_fp8(**{**asked, name: asked[name].detach()}), want)


@pytest.mark.parametrize("name", ("a_scales", "b_scales"))
def test_a_tangent_is_refused(inputs, name):
    with fwd.dual_level():
        asked = {**inputs, name: fwd.make_dual(inputs[name], torch.ones_like(inputs[name]))}
        with pytest.raises(ValueError, match="tangent"):
            dsa_amd.matmul_fp8(**asked)
