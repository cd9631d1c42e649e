"""The norm's gradient beside hooks of saved tensors, which may give back an equal tensor
that is laid out in another way."""
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


def make(shape, dtype, seed):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


def turned(t):
    """Columns next to each other instead of rows; of a single dimension, every second element."""
    if t.dim() > 1:
        return t.transpose(0, -1).contiguous().transpose(0, -1)
    return torch.stack([t, t], -1)[:, 0]


def spaced(t):
    return torch.cat([t, t], -1)[..., :t.shape[-1]]


def uneven(t):
    """Rows of a third dimension that follow each other at no even distance."""
    return torch.cat([t, t[:, :1]], 1)[:, :-1] if t.dim() > 2 else t


def away(t):
    return t.cpu()


def back(t):
    return t.cuda()


def negated(t):
    return torch._neg_view(-t)


@pytest.mark.parametrize("eps", [1e-6, 1])  # a whole number: the Python path
@pytest.mark.parametrize("dtype", [BF, FULL])
@pytest.mark.parametrize("pack, unpack", [(turned, lambda t: t), (spaced, lambda t: t), (uneven, lambda t: t), (away, back),
                                          (negated, lambda t: t)])
def test_saved_tensors_may_be_laid_out_otherwise(pack, unpack, dtype, eps):
    base = [make((4, 3, 520), dtype, 0), make(520, dtype, 1), make((4, 3, 520), dtype, 2)]
    given = [make((4, 3, 520), dtype, 3 + i) for i in range(2)]

    def step(residual):
        x, w, r = (t.clone().requires_grad_() for t in base)
        if residual:
            return torch.autograd.grad(dsa_amd.rms_norm(x, w, r, eps=eps), (x, w, r), given)
        return torch.autograd.grad(dsa_amd.rms_norm(x, w, eps=eps), (x, w), given[0])

    for residual in (False, True):
        want = step(residual)
        with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
            got = step(residual)
        for a, b in zip(got, want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("eps", [1e-6, 1])
@pytest.mark.parametrize("unpack", [lambda t: t.cpu(), lambda t: t.double(), lambda t: t[..., :-1], lambda t: t[None]])
def test_another_tensor_is_refused(unpack, eps):
    x, w = make((4, 520), FULL, 0).requires_grad_(), make(520, FULL, 1).requires_grad_()
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
        y = dsa_amd.rms_norm(x, w, eps=eps)
        with pytest.raises(RuntimeError, match="came back"):
            y.sum().backward()


class _Nothing(torch.autograd.Function):
    """A function that gives its inputs no gradient."""

    @staticmethod
    def forward(ctx, *tensors):
        return tensors[0].sum()

    @staticmethod
    def backward(ctx, grad):
        return (None,) * len(ctx.needs_input_grad)


@pytest.mark.parametrize("eps", [1e-6, 1])
@pytest.mark.parametrize("outputs", [(0,), (1,), (0, 1)])
def test_without_any_gradient(outputs, eps):
    """Behind a function that gives none the gradients are zeros."""
    x, w, r = make((4, 520), FULL, 0).requires_grad_(), make(520, FULL, 1).requires_grad_(), make((4, 520), FULL, 2).requires_grad_()
    out = dsa_amd.rms_norm(x, w, r, eps=eps)
    _Nothing.apply(*(out[i] for i in outputs)).backward()
    assert not x.grad.any() and not w.grad.any() and not r.grad.any()
    if outputs == (0,):
        w.grad = None
        _Nothing.apply(dsa_amd.rms_norm(x.detach(), w, eps=eps)).backward()
        assert w.grad.shape == (520,) and not w.grad.any()


@pytest.mark.parametrize("eps", [1e-6, 1])
def test_a_row_without_leading_dimensions(eps):
    x, w, g = make((1, 520), FULL, 0), make(520, FULL, 1), make((1, 520), FULL, 2)
    leaves = [x[0].clone().requires_grad_(), w.clone().requires_grad_(), x[0].clone().requires_grad_()]
    y, h = dsa_amd.rms_norm(*leaves, eps=eps)
    got = torch.autograd.grad((y, h), leaves, (g[0], g[0]))
    leaves = [x.clone().requires_grad_(), w.clone().requires_grad_(), x.clone().requires_grad_()]
    want = torch.autograd.grad(dsa_amd.rms_norm(*leaves, eps=eps), leaves, (g, g))
    for a, b in zip(got, want):
        assert torch.equal(a, b.view(a.shape))
