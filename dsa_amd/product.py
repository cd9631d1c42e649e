"""Products with 8-bit weights (no reference counterpart: the reference takes
``q`` and ``kv`` as given, README.md:19-21).

A layer's projections around the attention, with weights in e4m3 and a scale
for each block of 128 by 128: of the residual stream
(:func:`dsa_amd.rms_norm_fp8`) to the query and cache latents, of the query
latent to the heads, and of the heads' outputs (:func:`dsa_amd.quantize_fp8`)
back to the stream.  ``csrc/product.hip``; there is no CPU path.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from .api import _fast_layer, _on_device
from .norm import SCALE_BLOCK, _derivatives
from .rotary import DTYPES


def matmul_fp8(a, a_scales, b, b_scales, *, dtype=torch.bfloat16):
    """``a [..., K]`` times ``b [N, K]`` transposed: ``[..., N]``, where both are 8-bit
    codes (float8_e4m3fn) that stand for ``codes * scales``:

    * ``a_scales`` fp32 ``[..., ceil(K / 128)]``, one for each 128 of a row (as
      :func:`dsa_amd.rms_norm_fp8` and :func:`dsa_amd.quantize_fp8` give them);
    * ``b_scales`` fp32 ``[ceil(N / 128), ceil(K / 128)]``, one for each 128 by 128.

    The products of 128 are summed in 32 bits, multiplied by the product of their two
    scales (in 32 bits too: it has to be in their range), summed in 32 bits and rounded
    once to ``dtype`` (bfloat16, float16 or float32).  For the 16-bit ones the matrix
    cores cut each product to 2^-13 of the largest of eight neighbours (an error of
    1.5e-5 of a sum's size was measured); for float32
    they are whole, at half the rate.  The same inputs give the same
    bits.  K is a multiple of 16 below 2^20.  All inputs are contiguous, the codes
    16-byte aligned.  The output is a fresh tensor, and nothing synchronises.  No gradient
    is recorded, and as with :func:`dsa_amd.rms_norm_fp8` no input may require one while
    gradients are enabled, or carry a forward-mode tangent."""
    fast = _fast_layer()
    if fast is not None:  # checked, allocated and launched in C++ (None: not taken)
        taken = fast.matmul_fp8(a, a_scales, b, b_scales, dtype)
        if taken is not None:
            if type(taken) is int:
                _lib.check(taken, "dsa_matmul_fp8")
            return taken
    if not all(isinstance(t, torch.Tensor) for t in (a, a_scales, b, b_scales)):
        raise ValueError("a, a_scales, b and b_scales must be tensors")
    if a.dim() < 1 or b.dim() != 2 or a.shape[-1] != b.shape[1]:
        raise ValueError("expected a[..., K] and b[N, K]")
    columns, inner = b.shape
    if inner <= 0 or inner % 16 or inner >= 1 << 20 or not 0 < columns <= 1 << 24 or a.numel() > inner << 24 or (
            a.numel() // inner * columns > 1 << 37):
        raise ValueError("K must be a positive multiple of 16 below 2^20, N in [1, 2^24], and there be at most 2^24 rows and "
                         f"2^37 outputs (got {inner}, {columns} and {list(a.shape[:-1])})")
    blocks = -(-inner // SCALE_BLOCK)
    if a_scales.shape != (*a.shape[:-1], blocks) or b_scales.shape != (-(-columns // SCALE_BLOCK), blocks):
        raise ValueError(f"expected a_scales[..., {blocks}] and b_scales[{-(-columns // SCALE_BLOCK)}, {blocks}]")
    device = a.device
    if device.type != "cuda" or torch.version.hip is None or any(
            t.device != device or not t.is_contiguous() for t in (a, a_scales, b, b_scales)) or a.is_neg() or b.is_neg():
        raise ValueError("all inputs must be contiguous and on the same ROCm GPU")
    e4m3 = torch.float8_e4m3fn
    if a.dtype != e4m3 or b.dtype != e4m3 or a_scales.dtype != torch.float32 or b_scales.dtype != torch.float32:
        raise ValueError("a and b must be float8_e4m3fn, their scales float32")
    if dtype not in DTYPES:
        raise ValueError("dtype must be torch.bfloat16, torch.float16 or torch.float32")
    if any(_derivatives(a, a_scales, b, b_scales)):
        raise ValueError("matmul_fp8 records no gradient and no forward-mode tangent: call it without them (torch.no_grad)")
    a_scales, b_scales = a_scales.resolve_neg(), b_scales.resolve_neg()
    out = torch.empty((*a.shape[:-1], columns), device=device, dtype=dtype)
    if out.numel() == 0:
        return out
    args = _lib.DsaProductArgs()
    args.a, args.a_scales, args.b, args.b_scales = a.data_ptr(), a_scales.data_ptr(), b.data_ptr(), b_scales.data_ptr()
    args.out, args.dtype = out.data_ptr(), DTYPES[dtype]
    args.M, args.N, args.K = a.numel() // inner, columns, inner
    lib = _lib.load()
    with _on_device(device):
        rc = lib.dsa_matmul_fp8(ctypes.byref(args), torch._C._cuda_getCurrentRawStream(device.index))
    if rc:
        _lib.check(rc, "dsa_matmul_fp8")
    return out
