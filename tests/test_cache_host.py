"""Host contract of the paged cache's operators (rotary positions, block
tables, cache row writes): refusals that need no device, the C ABI's argument
checks, the frequencies, and the header against its binding."""
import ctypes
import math
import re
from pathlib import Path

import pytest
import torch

import dsa_amd
from dsa_amd import _lib

HEADER = Path(__file__).resolve().parents[1] / "include" / "dsa_mi355x_cache.h"


def test_header_and_binding_agree():
    text = re.sub(r"/\*.*?\*/", "", HEADER.read_text(), flags=re.S)
    declared = sorted(set(re.findall(r"\b(dsa_[a-z_]+)\s*\(", text)))
    assert declared == sorted(_lib.CACHE_SIGNATURES)
    lib = _lib.load()
    for name in declared:
        assert hasattr(lib, name), name


def test_struct_layouts(tmp_path):
    """Field offsets of the argument structs as a C compiler lays them out."""
    import subprocess

    structs = {"dsa_rotary_args": _lib.DsaRotaryArgs, "dsa_write_args": _lib.DsaWriteArgs,
               "dsa_shared_args": _lib.DsaSharedArgs}
    lines = [f'printf("%s %s %zu\\n", "{n}", "{f[0]}", offsetof({n}, {f[0]}));' for n, s in structs.items()
             for f in s._fields_]
    lines += [f'printf("%s sizeof %zu\\n", "{n}", sizeof({n}));' for n in structs]
    src = tmp_path / "layout.c"
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "dsa_mi355x.h"\n#include "dsa_mi355x_cache.h"\n'
                   "int main(void) {" + "\n".join(lines) + "return 0;}\n")
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", f"-I{HEADER.parent}", str(src), "-o", str(exe)], check=True)
    for line in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines():
        name, field, value = line.split()
        struct = structs[name]
        assert int(value) == (ctypes.sizeof(struct) if field == "sizeof" else getattr(struct, field).offset), line


# ------------------------------------------------------------ frequencies

def test_plain_frequencies():
    f = dsa_amd.rotary_frequencies(64)
    assert f.dtype == torch.float64 and f.shape == (32,)
    for i in (0, 1, 17, 31):
        assert f[i].item() == pytest.approx(10000.0 ** (-2 * i / 64), rel=1e-15)
    linear = dsa_amd.rotary_frequencies(64, scaling="linear", factor=8.0)
    assert torch.equal(linear, f / 8.0)


def test_yarn_frequencies():
    """Pairs that turn often keep their frequency, pairs that turn less than
    once are stretched whole, and the ones between lie between, in order."""
    f = dsa_amd.rotary_frequencies(64)
    y = dsa_amd.rotary_frequencies(64, scaling="yarn", factor=40.0, original_length=4096)
    turns = f * 4096 / (2 * math.pi)
    ratio = f / y
    # the borders are rounded outward to whole pairs: 32 turns lie at pair 10.45, 1 turn at 22.51
    assert torch.allclose(ratio[:11], torch.ones(11, dtype=torch.float64), rtol=1e-15)
    assert torch.allclose(ratio[23:], torch.full((9,), 40.0, dtype=torch.float64), rtol=1e-15)
    assert turns[10] > 32 > turns[11] and turns[22] > 1 > turns[23]
    keep = 1 - (torch.arange(11, 23, dtype=torch.float64) - 10) / 13
    assert torch.allclose(y[11:23], f[11:23] * keep + f[11:23] / 40 * (1 - keep), rtol=1e-14)
    assert (y[1:] < y[:-1]).all()


@pytest.mark.parametrize("kw", [dict(dim=63), dict(dim=0), dict(dim=514), dict(dim=64, theta=1.0),
                                dict(dim=64, theta=math.inf), dict(dim=64, scaling="ntk"), dict(dim=64, factor=0.0),
                                dict(dim=64, scaling="yarn", beta_fast=1.0, beta_slow=2.0),
                                dict(dim=64, scaling="yarn", original_length=0), dict(dim=64.0)])
def test_frequency_refusals(kw):
    with pytest.raises(ValueError):
        dsa_amd.rotary_frequencies(**kw)


# ------------------------------------------------------------ refusals on the host

def test_cpu_tensors_are_refused():
    f = dsa_amd.rotary_frequencies(64)
    x = torch.zeros(2, 4, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="ROCm GPU"):
        dsa_amd.rotary(x, torch.zeros(2, dtype=torch.int32), f)
    with pytest.raises(ValueError, match="ROCm GPU"):
        dsa_amd.extend_block_table(torch.zeros(2, 4, dtype=torch.int32), *(torch.zeros(2, dtype=torch.int32),) * 3, 16, 4)
    with pytest.raises(ValueError, match="ROCm GPU"):
        dsa_amd.write_kv_rows(torch.zeros(2, 512, dtype=torch.bfloat16), torch.zeros(2, 64, dtype=torch.bfloat16),
                              torch.zeros(2, dtype=torch.int32), torch.zeros(4, 1, 512, dtype=torch.bfloat16),
                              torch.zeros(4, 1, 64, dtype=torch.bfloat16))


@pytest.mark.parametrize("x", [None, torch.zeros(64), torch.zeros(2, 64), torch.zeros(1, 1, 1, 2, 64)])
def test_rotary_shapes_are_refused(x):
    with pytest.raises(ValueError, match="tokens, H, D"):
        dsa_amd.rotary(x, torch.zeros(2, dtype=torch.int32), dsa_amd.rotary_frequencies(64))


@pytest.mark.parametrize("table, block, most", [
    (torch.zeros(4, dtype=torch.int32), 16, 4), (torch.zeros(0, 4, dtype=torch.int32), 16, 4),
    (torch.zeros(2, 4, dtype=torch.int32), 0, 4), (torch.zeros(2, 4, dtype=torch.int32), 16.0, 4),
    (torch.zeros(2, 4, dtype=torch.int32), 16, -1), (torch.zeros(4097, 1, dtype=torch.int32), 16, 4)])
def test_table_arguments_are_refused(table, block, most):
    v = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError):
        dsa_amd.extend_block_table(table, v, v, v, block, most)


def test_write_shapes_are_refused():
    bf = torch.bfloat16
    kv, kr, slots = torch.zeros(2, 512, dtype=bf), torch.zeros(2, 64, dtype=bf), torch.zeros(2, dtype=torch.int32)
    pool, rope = torch.zeros(4, 16, 1, 512, dtype=bf), torch.zeros(4, 16, 1, 64, dtype=bf)
    rows = torch.zeros(4, 16, 1, 656, dtype=torch.uint8)
    for args in [(kv[:, :511], kr, slots, pool, rope), (kv, kr[:1], slots, pool, rope), (kv, kr, slots, pool, None),
                 (kv, kr, slots, rows, rope), (kv, kr, slots, pool[..., :511], rope), (kv, kr, slots, pool, rope[:3]),
                 (kv, kr, slots, rows[..., :655]), (kv[None], kr[None], slots, pool, rope)]:
        with pytest.raises(ValueError):
            dsa_amd.write_kv_rows(*args)


# ------------------------------------------------------------ C argument checks

def _rotary_args(**kw):
    a = _lib.DsaRotaryArgs()
    a.x = a.out = a.positions = a.frequencies = 4096
    a.groups = a.tokens = 1
    a.heads, a.width, a.start, a.dim, a.magnitude = 2, 64, 0, 64, 1.0
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw", [dict(x=None), dict(out=None), dict(positions=None), dict(frequencies=None), dict(dtype=3),
                                dict(dim=63), dict(dim=0), dict(dim=1024, width=1024), dict(start=1), dict(start=-1),
                                dict(tokens=0), dict(groups=0), dict(heads=0), dict(width=0), dict(x=4097),
                                dict(frequencies=4100), dict(positions=4100, positions_64=1), dict(magnitude=math.inf),
                                dict(groups=1 << 31, tokens=1 << 31), dict(dtype=2, out=4098)])
def test_c_rotary_refuses(kw):
    lib = _lib.load()
    assert lib.dsa_rotary(ctypes.byref(_rotary_args(**kw)), None) < 0
    assert lib.dsa_last_error()


@pytest.mark.parametrize("kw", [dict(kv=None), dict(k_rope=None), dict(slots=None), dict(cache=None), dict(rope_cache=None),
                                dict(frequencies=4096, positions=None), dict(kv_format=2), dict(kv_format=1),
                                dict(tokens=0), dict(cache_rows=0), dict(kv_stride=516), dict(rope_stride=65),
                                dict(kv=4104), dict(k_rope=4098), dict(magnitude=math.nan)])
def test_c_write_refuses(kw):
    lib = _lib.load()
    a = _lib.DsaWriteArgs()
    a.kv = a.k_rope = a.slots = a.cache = a.rope_cache = 4096
    a.tokens, a.cache_rows, a.kv_stride, a.rope_stride, a.magnitude = 1, 4, 512, 64, 1.0
    for k, v in kw.items():
        setattr(a, k, v)
    assert lib.dsa_write_kv_rows(ctypes.byref(a), None) < 0
    assert lib.dsa_last_error()


@pytest.mark.parametrize("at, value", [(0, None), (1, None), (2, None), (3, None), (4, None), (5, None), (6, None),
                                       (7, None), (8, None), (9, 0), (9, 4097), (10, 0), (11, 0), (12, -1), (13, -1)])
def test_c_table_refuses(at, value):
    lib = _lib.load()
    args = [4096] * 9 + [2, 4, 16, 3, 8, None]
    args[at] = value
    assert lib.dsa_extend_block_table(*args) < 0
    assert lib.dsa_last_error()


def _shared_args(**kw):
    a = _lib.DsaSharedArgs()
    for name in ("q", "kv", "q_rope", "k_rope", "lengths", "out", "out_max", "out_sum", "workspace"):
        setattr(a, name, 4096)
    a.workspace_bytes, a.num_cus = 1 << 40, 256
    a.B, a.SQ, a.H, a.L, a.prefix = 3, 2, 16, 128, 64
    for k, v in kw.items():
        setattr(a, k, v)
    return a


SIZES = [dict(B=0), dict(SQ=0), dict(H=0), dict(H=24), dict(L=0), dict(L=1 << 25, prefix=0), dict(prefix=-1),
         dict(prefix=129), dict(num_cus=-1), dict(num_cus=4097), dict(B=1 << 20, SQ=1 << 10, H=128)]


@pytest.mark.parametrize("kw", SIZES + [
    dict(q=None), dict(kv=None), dict(q_rope=None), dict(k_rope=None), dict(lengths=None), dict(out=None),
    dict(out_max=None), dict(out_sum=None), dict(workspace=None), dict(q=4104), dict(kv=4104), dict(k_rope=4104),
    dict(out=4104), dict(lengths=4098), dict(workspace=4112), dict(kv_format=2), dict(scale=-1.0), dict(scale=math.nan),
    dict(block_table=4096), dict(block_table=4096, block_size=16, max_blocks=7, num_blocks=9),
    dict(block_table=4096, block_size=16, max_blocks=8, num_blocks=0), dict(workspace_bytes=1 << 16),
    dict(block_table=4096, block_size=16, max_blocks=8, num_blocks=1 << 21)])
def test_c_shared_refuses(kw):
    lib = _lib.load()
    assert lib.dsa_fwd_shared(ctypes.byref(_shared_args(**kw)), None) < 0
    assert lib.dsa_last_error()


@pytest.mark.parametrize("kw", SIZES)
def test_c_shared_workspace_refuses(kw):
    assert _lib.load().dsa_fwd_shared_ws_bytes(ctypes.byref(_shared_args(**kw))) < 0


def test_c_shared_workspace():
    """Grows with the batch and the workgroups; a row of a piece is 512 + 2 floats."""
    lib = _lib.load()
    size = lambda **kw: lib.dsa_fwd_shared_ws_bytes(ctypes.byref(_shared_args(**kw)))  # noqa: E731
    assert size(B=1, SQ=1, prefix=0) == 256 + 2 * 256 * 16 * 514 * 4
    assert size(B=1, SQ=64, prefix=0) == 256 + 2 * 256 * 128 * 514 * 4
    # 4 items of 128 stacked rows, 32 of 16 own ones, and a cut for each workgroup
    assert size(B=32, SQ=1) == 512 + ((4 + 256) * 128 + (32 + 256) * 16) * 514 * 4
    assert size(B=32, SQ=1, num_cus=8) < size(B=32, SQ=1) < size(B=4096, SQ=1)


def test_shared_inputs_are_refused():
    bf = torch.bfloat16
    q, qr, lengths = torch.zeros(2, 1, 16, 512, dtype=bf), torch.zeros(2, 1, 16, 64, dtype=bf), torch.zeros(2, 1, dtype=torch.int32)
    kv, kr = torch.zeros(2, 8, 1, 512, dtype=bf), torch.zeros(2, 8, 1, 64, dtype=bf)
    for args in [(q, kv, qr, kr, lengths), (q, kv, qr, None, lengths), (None, kv, qr, kr, lengths),
                 (q, kv, qr, kr, [8, 8]), (q[0], kv, qr, kr, lengths), (q, kv[..., :511], qr, kr, lengths),
                 (q[:, :, :8], kv, qr[:, :, :8], kr, lengths), (q, kv, qr, kr, lengths, 9), (q, kv, qr, kr, lengths, True)]:
        with pytest.raises(ValueError):
            dsa_amd.forward_shared(*args)
