"""Host contract of the norms, 8-bit products and drafted trees: the header against
its binding, the C ABI's argument checks, and refusals that need no device."""
import ctypes
import math
import re
import subprocess
from pathlib import Path

import pytest
import torch

import dsa_amd
from dsa_amd import _lib

HEADER = Path(__file__).resolve().parents[1] / "include" / "dsa_mi355x_layer.h"


def test_header_and_binding_agree():
    text = re.sub(r"/\*.*?\*/", "", HEADER.read_text(), flags=re.S)
    declared = sorted(set(re.findall(r"\b(dsa_[a-z0-9_]+)\s*\(", text)))
    assert declared == sorted(_lib.LAYER_SIGNATURES)
    lib = _lib.load()
    for name in declared:
        assert hasattr(lib, name), name


def test_struct_layouts(tmp_path):
    """Field offsets of the argument structs as a C compiler lays them out."""
    structs = {"dsa_norm_args": _lib.DsaNormArgs, "dsa_norm_grad_args": _lib.DsaNormGradArgs,
               "dsa_product_args": _lib.DsaProductArgs, "dsa_tree_args": _lib.DsaTreeArgs}
    lines = [f'printf("%s %s %zu\\n", "{n}", "{f[0]}", offsetof({n}, {f[0]}));' for n, s in structs.items()
             for f in s._fields_]
    lines += [f'printf("%s sizeof %zu\\n", "{n}", sizeof({n}));' for n in structs]
    src = tmp_path / "layout.c"
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "dsa_mi355x.h"\n#include "dsa_mi355x_layer.h"\n'
                   "int main(void) {" + "\n".join(lines) + "return 0;}\n")
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", f"-I{HEADER.parent}", str(src), "-o", str(exe)], check=True)
    for line in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines():
        name, field, value = line.split()
        struct = structs[name]
        assert int(value) == (ctypes.sizeof(struct) if field == "sizeof" else getattr(struct, field).offset), line
    assert (_lib.BF16, _lib.F16, _lib.F32) == (0, 1, 2)


def _fill(a, /, **kw):
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def _norm_args(**kw):
    a = _lib.DsaNormArgs()
    a.x = a.weight = a.out = a.scales = 4096
    a.rows, a.x_stride, a.dim, a.eps = 2, 512, 512, 1e-6
    return _fill(a, **kw)


NORM = [dict(x=None), dict(out=None), dict(residual=4096), dict(dtype=3), dict(dim=0), dict(dim=16385), dict(rows=0),
        dict(x_stride=-1), dict(x_stride=1 << 41), dict(eps=-1.0), dict(eps=math.nan), dict(eps=math.inf), dict(x=4097),
        dict(weight=4097), dict(weight=4098, weight_f32=1), dict(x=4098, dtype=2), dict(rows=1 << 41),
        dict(rows=1 << 40, x_stride=1 << 40), dict(residual=4097, sum=4096)]


@pytest.mark.parametrize("kw", NORM + [dict(weight=None), dict(out=4097)])
def test_c_norm_refuses(kw):
    lib = _lib.load()
    assert lib.dsa_rms_norm(ctypes.byref(_norm_args(**kw)), None) < 0
    assert lib.dsa_last_error()


@pytest.mark.parametrize("kw", NORM + [dict(scales=None), dict(dim=520), dict(out=4104), dict(scales=4098),
                                       dict(weight=None, residual=4096, sum=4096)])
def test_c_norm_fp8_refuses(kw):
    lib = _lib.load()
    assert lib.dsa_rms_norm_fp8(ctypes.byref(_norm_args(**kw)), None) < 0
    assert lib.dsa_last_error()


def _grad_args(**kw):
    a = _lib.DsaNormGradArgs()
    a.h = a.inverse = a.weight = a.grad_out = a.grad_in = a.grad_weight = a.workspace = 4096
    a.rows, a.h_stride, a.dim, a.workspace_bytes = 2, 512, 512, 1 << 30
    return _fill(a, **kw)


@pytest.mark.parametrize("kw", [dict(h=None), dict(inverse=None), dict(weight=None), dict(grad_out=None), dict(grad_in=None),
                                dict(workspace=None), dict(workspace_bytes=100), dict(workspace=4104), dict(dtype=-1),
                                dict(dim=0), dict(rows=0), dict(h=4097), dict(grad_sum=4097), dict(inverse=4098),
                                dict(grad_weight=4098, weight_f32=1), dict(h_stride=-8)])
def test_c_norm_grad_refuses(kw):
    lib = _lib.load()
    assert lib.dsa_rms_norm_grad(ctypes.byref(_grad_args(**kw)), None) < 0
    assert lib.dsa_last_error()
    assert lib.dsa_rms_norm_grad_ws_bytes(0, 512) < 0 and lib.dsa_rms_norm_grad_ws_bytes(5, 16385) < 0
    assert 0 < lib.dsa_rms_norm_grad_ws_bytes(1, 512) <= lib.dsa_rms_norm_grad_ws_bytes(1 << 40, 512) <= 1 << 26


def _product_args(**kw):
    a = _lib.DsaProductArgs()
    a.a = a.a_scales = a.b = a.b_scales = a.out = 4096
    a.M, a.N, a.K = 5, 100, 256
    return _fill(a, **kw)


@pytest.mark.parametrize("kw", [dict(M=0), dict(N=0), dict(K=0), dict(K=8), dict(K=250), dict(K=1 << 20), dict(M=(1 << 24) + 1),
                                dict(N=(1 << 24) + 1), dict(M=1 << 19, N=(1 << 18) + 1), dict(dtype=3), dict(a=None),
                                dict(a_scales=None), dict(b=None), dict(b_scales=None), dict(out=None),
                                dict(a=4104), dict(b=4104), dict(a_scales=4098), dict(b_scales=4098), dict(out=4097),
                                dict(out=4098, dtype=2)])
def test_c_product_refuses(kw):
    lib = _lib.load()
    assert lib.dsa_matmul_fp8(ctypes.byref(_product_args(**kw)), None) < 0
    assert lib.dsa_last_error()
    assert lib.dsa_matmul_fp8(None, None) < 0


def _tree_args(**kw):
    a = _lib.DsaTreeArgs()
    for name in ("q", "kv", "q_rope", "k_rope", "lengths", "out", "out_max", "out_sum", "workspace"):
        setattr(a.shared, name, 4096)
    a.shared.workspace_bytes, a.shared.num_cus = 1 << 40, 256
    a.shared.B, a.shared.SQ, a.shared.H, a.shared.L, a.shared.prefix = 3, 2, 16, 128, 64
    a.tree, a.words = 4096, 1
    for k, v in kw.items():
        setattr(a if k in ("tree", "words") else a.shared, k, v)
    return a


@pytest.mark.parametrize("kw", [dict(tree=None), dict(tree=4098), dict(words=0), dict(words=65), dict(q=None), dict(H=24),
                                dict(L=0), dict(workspace_bytes=100), dict(scale=-1.0), dict(lengths=4097)])
def test_c_tree_refuses(kw):
    lib = _lib.load()
    assert lib.dsa_fwd_tree(ctypes.byref(_tree_args(**kw)), None) < 0
    assert lib.dsa_last_error()
    assert lib.dsa_fwd_tree_ws_bytes(None) < 0 and lib.dsa_fwd_tree_ws_bytes(ctypes.byref(_tree_args(H=24))) < 0
    args = _tree_args()
    assert lib.dsa_fwd_tree_ws_bytes(ctypes.byref(args)) == lib.dsa_fwd_shared_ws_bytes(ctypes.byref(args.shared)) > 0


@pytest.mark.parametrize("at, value", [(0, None), (1, None), (2, None), (3, None), (0, 4098), (3, 4098), (4, 0), (4, (1 << 20) + 1),
                                       (5, 0), (5, 2049)])
def test_c_draft_tree_refuses(at, value):
    lib = _lib.load()
    args = [4096] * 4 + [2, 8, None]
    args[at] = value
    assert lib.dsa_draft_tree(*args) < 0
    assert lib.dsa_last_error()


def test_cpu_tensors_are_refused():
    x, w = torch.zeros(2, 128), torch.ones(128)
    i32 = lambda *shape: torch.zeros(shape, dtype=torch.int32)  # noqa: E731
    for call in (lambda: dsa_amd.rms_norm(x, w), lambda: dsa_amd.rms_norm_fp8(x, w), lambda: dsa_amd.quantize_fp8(x),
                 lambda: dsa_amd.matmul_fp8(x.to(torch.float8_e4m3fn), x[:, :1].contiguous(), x.to(torch.float8_e4m3fn),
                                            x[:1, :1].contiguous()),
                 lambda: dsa_amd.draft_tree(i32(2, 3), i32(2)),
                 lambda: dsa_amd.forward_tree(torch.zeros(2, 1, 16, 512).bfloat16(), torch.zeros(2, 8, 1, 512).bfloat16(),
                                              torch.zeros(2, 1, 16, 64).bfloat16(), torch.zeros(2, 8, 1, 64).bfloat16(), i32(2),
                                              i32(2, 1, 1))):
        with pytest.raises(ValueError, match="ROCm GPU"):
            call()
    for bad in (None, [1.0], torch.zeros(())):
        with pytest.raises(ValueError):
            dsa_amd.rms_norm(bad, w)
        with pytest.raises(ValueError):
            dsa_amd.quantize_fp8(bad)
