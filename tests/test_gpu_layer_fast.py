"""The host fast path of the norms, products and drafted trees (dsa_amd/_fast_layer*.so,
_fast_cache*.so): the same results as the Python path, and None for whatever that
refuses or does besides."""
import sys

import pytest
import torch

import dsa_amd
from dsa_amd import api

pytestmark = pytest.mark.gpu

BF, E4M3 = torch.bfloat16, torch.float8_e4m3fn


@pytest.fixture(scope="module")
def fast():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm GPU")
    module = api._fast_layer()
    assert module is not None, "the fast path module is built by dsa_amd.build"
    return module


@pytest.fixture
def slow(fast, monkeypatch):
    """Both ways of a call: as it is, and in Python."""
    def both(module, call):
        first = call()
        with monkeypatch.context() as m:
            for name in ("_fast_layer", "_fast_cache"):
                if hasattr(sys.modules["dsa_amd." + module], name):
                    m.setattr(sys.modules["dsa_amd." + module], name, lambda: None)
            second = call()
        return first, second
    return both


def make(*shape, dtype=BF, seed=0):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


def i32(v):
    return torch.tensor(v, dtype=torch.int32).cuda()


def same(a, b):
    a, b = (x if isinstance(x, tuple) else (x,) for x in (a, b))
    assert len(a) == len(b)
    for x, y in zip(a, b):
        assert x.dtype == y.dtype and x.shape == y.shape and x.stride() == y.stride() and x.requires_grad == y.requires_grad
        bits = torch.uint8 if x.dtype == E4M3 else x.dtype
        assert torch.equal(x.view(bits), y.view(bits))


def test_norms_are_equal(slow):
    wide = make(4, 3, 700)
    for x in (make(5, 512), wide[..., :640], wide[..., 3:515], make(7, dtype=torch.float16), wide[:, 0, :640]):
        w, r = make(x.shape[-1], dtype=x.dtype, seed=1), make(*x.shape, dtype=x.dtype, seed=2)
        for args in ((x, w), (x, w, r), (x, w.float(), r)):
            same(*slow("norm", lambda: dsa_amd.rms_norm(*args, eps=0.01)))
            if x.shape[-1] % 16 == 0:
                for pow2 in (True, False):
                    same(*slow("norm", lambda: dsa_amd.rms_norm_fp8(*args, pow2_scales=pow2)))
                    same(*slow("norm", lambda: dsa_amd.quantize_fp8(x, pow2_scales=pow2)))


@pytest.mark.parametrize("which", [(0,), (1,), (2,), (0, 1), (0, 2), (1, 2), (0, 1, 2)])
@pytest.mark.parametrize("outputs", [(0,), (1,), (0, 1)])
def test_gradients_are_equal(slow, which, outputs):
    base = [make(9, 520, dtype=torch.float32), make(520, dtype=torch.float32, seed=1), make(9, 520, dtype=torch.float32, seed=2)]
    given = [make(9, 520, dtype=torch.float32, seed=3 + i) for i in range(2)]

    def call():
        leaves = [t.clone().requires_grad_(i in which) for i, t in enumerate(base)]
        out = dsa_amd.rms_norm(*leaves)
        assert all(t.requires_grad and not t.is_leaf for t in out)
        grads = torch.autograd.grad([out[i] for i in outputs], [leaves[i] for i in which], [given[i] for i in outputs])
        return (*(t.detach() for t in out), *grads)

    same(*slow("norm", call))


def test_gradients_refuse_the_same(slow):
    def twice():
        x = make(2, 64).requires_grad_()
        g, = torch.autograd.grad(dsa_amd.rms_norm(x, make(64)).square().sum(), x, create_graph=True)
        with pytest.raises(RuntimeError, match="once_differentiable"):
            g.sum().backward()

    def written():
        x = make(2, 64).requires_grad_()
        y, h = dsa_amd.rms_norm(x, make(64), make(2, 64))
        with torch.no_grad():
            h.add_(1.0)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.sum().backward()

    for call in (twice, written):
        slow("norm", call)


def test_a_training_step_accumulates(slow):
    def call():
        model = [torch.nn.Parameter(make(640, dtype=torch.float32, seed=i)) for i in range(3)]
        x = make(6, 640, dtype=torch.float32, seed=9)
        y, stream = dsa_amd.rms_norm(x, model[0]), x
        for w in model[1:]:
            y, stream = dsa_amd.rms_norm(y, w, stream)
        (y * stream).sum().backward()
        return tuple(w.grad for w in model)

    same(*slow("norm", call))


def test_products_and_trees_are_equal(slow):
    codes, scales = dsa_amd.quantize_fp8(make(2, 5, 272))
    b, bs = make(200, 272).to(E4M3), torch.rand(2, 3).cuda()
    for dtype in (BF, torch.float16, torch.float32):
        same(*slow("product", lambda: dsa_amd.matmul_fp8(codes, scales, b, bs, dtype=dtype)))
    parents, lengths = i32([[-1, 0, 0, 7], [-1, -1, 1, -2]]), i32([20, 9])
    same(*slow("tree", lambda: dsa_amd.draft_tree(parents, lengths)))
    tree = dsa_amd.draft_tree(parents, lengths)[0]
    q, qr, kv, kr = make(2, 4, 16, 512), make(2, 4, 16, 64), make(2, 32, 1, 512), make(2, 32, 1, 64)
    rows, table = dsa_amd.quantize_kv_fp8(kv, kr), i32([[1, 0], [0, 1]])
    same(*slow("shared", lambda: dsa_amd.forward_tree(q, kv, qr, kr, lengths, tree, 5)))
    same(*slow("shared", lambda: dsa_amd.forward_tree(q, rows, qr, None, lengths, tree, scale=0.05, block_table=table)))


def test_declines(fast):
    """Declined before anything is allocated."""
    x, w = make(4, 512), make(512)
    codes, scales = dsa_amd.quantize_fp8(x)
    b, bs = make(100, 512).to(E4M3), torch.rand(1, 4).cuda()
    q, qr, kv, kr, lengths = make(2, 3, 16, 512), make(2, 3, 16, 64), make(2, 8, 1, 512), make(2, 8, 1, 64), i32([3, 4])
    tree, parents = torch.zeros(2, 3, 1, dtype=torch.int32).cuda(), i32([[-1, 0, 1], [-1, 0, 1]])
    off = torch.cat([codes.flatten()[:1].view(torch.uint8), codes.flatten().view(torch.uint8)]).view(E4M3)[1:].view(4, 512)
    good = {"rms_norm": (x, w, None, 1e-6), "rms_norm_fp8": (x, w, None, 1e-6, True), "quantize_fp8": (x, True),
            "matmul_fp8": (codes, scales, b, bs, BF), "draft_tree": (parents, lengths),
            "forward_tree": (q, kv, qr, kr, lengths, tree, 0, None, None)}
    norm = [{0: None}, {0: x.cpu()}, {0: x.double()}, {0: x[:, ::2]}, {0: x[:0]}, {1: None}, {1: w.cpu()}, {1: w.half()},
            {1: w[:511]}, {1: w[None]}, {2: x[:3]}, {2: x.float()}, {2: x.cpu()}, {2: 1}, {3: 1}, {3: -1.0}, {3: float("nan")},
            {3: None}, {0: make(2, 16400), 1: make(16400)}]
    bad = {"rms_norm": norm, "rms_norm_fp8": norm + [{4: None}, {4: 1}, {0: make(4, 520), 1: make(520)},
                                                     {0: x.clone().requires_grad_()}, {1: w.clone().requires_grad_()}],
           "quantize_fp8": [{0: None}, {0: x.cpu()}, {0: make(4, 520)}, {1: None}, {0: x.clone().requires_grad_()}],
           "matmul_fp8": [{0: None}, {0: codes.cpu()}, {0: codes.view(torch.uint8)}, {0: codes[:, :256]}, {0: off}, {0: codes[:0], 1: scales[:0]},
                          {1: scales[:3]}, {1: scales.double()}, {1: scales.t().contiguous().t()}, {2: b[:, :256]}, {2: b.cpu()},
                          {2: b[None]}, {3: bs[:, :3]}, {3: bs.half()}, {4: torch.float64}, {4: "bf16"}, {4: None}],
           "draft_tree": [{0: None}, {0: parents.cpu()}, {0: parents.long()}, {0: parents[0]}, {0: parents[:, :0]}, {1: lengths[:1]},
                          {1: lengths.long()}, {1: None}, {0: parents.t(), 1: i32([1, 2, 3])}],
           "forward_tree": [{0: None}, {0: q.float()}, {1: kv.cpu()}, {3: None}, {4: lengths.long()}, {4: lengths[:1]}, {5: None},
                            {5: tree[:, :2]}, {5: tree.long()}, {5: tree[..., :0]}, {5: tree.cpu()}, {6: 9}, {6: True}, {7: 0.0},
                            {8: tree}]}
    for name, args in good.items():
        call = getattr(api._fast_cache() if name in ("draft_tree", "forward_tree") else fast, name)
        assert call(*args) is not None and type(call(*args)) is not int
        for change in bad[name]:
            given = [change.get(i, a) for i, a in enumerate(args)]
            torch.cuda.synchronize()
            before = torch.cuda.memory_allocated()
            print(name, list(change), flush=True)
            assert call(*given) is None, (name, list(change))
            assert torch.cuda.memory_allocated() == before
