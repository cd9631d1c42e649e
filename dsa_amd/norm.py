"""Root-mean-square norms of a residual stream, and 8-bit codes with a scale for
each 128 values (no reference counterpart: the reference takes ``q`` and ``kv``
as given, README.md:19-21).

What stands in front of an attention layer's projections: :func:`rms_norm` in
16 or 32 bits, with the residual's addition and the gradients;
:func:`rms_norm_fp8` with an output for :func:`dsa_amd.matmul_fp8`; and
:func:`quantize_fp8`, which makes such codes of the attention's own output.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from .api import _fast_layer, _on_device
from .rotary import DTYPES, has_tangent

NORM_MAX_DIM = 16384
SCALE_BLOCK = 128


def _row_stride(t):
    """Elements between rows of the last dimension, or None where they are not evenly spaced."""
    lead = [(n, s) for n, s in zip(t.shape[:-1], t.stride()[:-1]) if n != 1]
    if not lead:
        return t.shape[-1]
    for (_, outer), (n, inner) in zip(lead, lead[1:]):
        if outer != n * inner:
            return None
    return lead[-1][1]


def _check_rows(t, name, shape, dtype, device):
    if not isinstance(t, torch.Tensor) or t.shape != shape or t.dtype != dtype or t.device != device:
        raise ValueError(f"{name} must have x's shape, type and device")


def _check(x, weight, residual, eps):
    if not isinstance(x, torch.Tensor) or x.dim() < 1:
        raise ValueError("x must be [..., dim]")
    device, dim = x.device, x.shape[-1]
    if device.type != "cuda" or torch.version.hip is None:
        raise ValueError("x must be on a ROCm GPU")
    if x.dtype not in DTYPES:
        raise ValueError("x must be bfloat16, float16 or float32")
    if not 1 <= dim <= NORM_MAX_DIM:
        raise ValueError(f"x's last dimension must be in [1, {NORM_MAX_DIM}] (got {dim})")
    if weight is not None:
        if not isinstance(weight, torch.Tensor) or weight.shape != (dim,) or weight.dtype not in (x.dtype, torch.float32):
            raise ValueError(f"weight must be [{dim}], of x's type or float32")
        if weight.device != device or not weight.is_contiguous():
            raise ValueError("weight must be contiguous and on x's device")
    if residual is not None:
        _check_rows(residual, "residual", x.shape, x.dtype, device)
    for t, name in ((x, "x"), (residual, "residual")):
        if t is not None and t.numel() > 0 and ((dim > 1 and t.stride(-1) != 1) or _row_stride(t) is None):
            raise ValueError(f"{name}'s last stride must be 1 and its rows evenly spaced")
    if isinstance(eps, bool) or not isinstance(eps, (int, float)):
        raise TypeError("eps must be a float")
    if not 0.0 <= eps <= 3.4028234663852886e38:
        raise ValueError("eps must be a finite 32-bit number, not negative")
    return dim


def _derivatives(*tensors):
    """Whether a gradient is to be recorded of some of them, and whether one carries a forward-mode tangent."""
    given = [t for t in tensors if t is not None]
    return torch.is_grad_enabled() and any(t.requires_grad for t in given), any(has_tangent(t) for t in given)


def _plain(*tensors):
    """Views whose sign is kept apart from their memory, as tensors that hold it."""
    return [t if t is None else t.resolve_neg() for t in tensors]


def _norm_args(x, weight, residual, eps, out, total):
    dim = x.shape[-1]
    args = _lib.DsaNormArgs()
    args.x, args.out = x.data_ptr(), out.data_ptr()
    args.rows, args.x_stride, args.dim, args.dtype = x.numel() // dim, _row_stride(x), dim, DTYPES[x.dtype]
    if weight is not None:
        args.weight, args.weight_f32 = weight.data_ptr(), weight.dtype == torch.float32
    if residual is not None:
        args.residual, args.residual_stride, args.sum = residual.data_ptr(), _row_stride(residual), total.data_ptr()
    args.eps = eps
    return args


def _launch(entry, args, device):
    with _on_device(device):
        rc = getattr(_lib.load(), entry)(ctypes.byref(args), torch._C._cuda_getCurrentRawStream(device.index))
    if rc:
        _lib.check(rc, entry)


def _norm(x, weight, residual, eps, keep):
    """y, the stream (x itself without a residual) and, to keep for the gradient, each row's inverse size."""
    y = torch.empty(x.shape, device=x.device, dtype=x.dtype)
    total = None if residual is None else torch.empty(x.shape, device=x.device, dtype=x.dtype)
    inverse = torch.empty(x.shape[:-1], device=x.device, dtype=torch.float32) if keep else None
    if x.numel() > 0:
        args = _norm_args(x, weight, residual, eps, y, total)
        if keep:
            args.inverse = inverse.data_ptr()
        _launch("dsa_rms_norm", args, x.device)
    return y, total, inverse


def _kept(t, shape, dtypes, device):
    """A tensor that was saved for the gradient.  Hooks of saved tensors may have put another
    in its place: equal, says their contract, but laid out in any way."""
    if t.shape != shape or t.dtype not in dtypes or t.device != device or t.layout != torch.strided:
        raise RuntimeError("rms_norm: a saved tensor came back with another shape, type or device")
    return t.resolve_neg()


class _RmsNorm(torch.autograd.Function):
    """Keeps the stream behind the addition and a number a row; the gradient of both summands is the same."""

    @staticmethod
    def forward(ctx, x, weight, residual, eps):
        y, total, inverse = _norm(x, weight, residual, eps, True)
        ctx.save_for_backward(x if total is None else total, weight, inverse)
        return y if total is None else (y, total)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_y, grad_total=None):
        shape, dtype, device = grad_y.shape, grad_y.dtype, grad_y.device
        h, weight, inverse = ctx.saved_tensors
        h = _kept(h, shape, (dtype,), device)
        if h.numel() > 0 and ((h.shape[-1] > 1 and h.stride(-1) != 1) or _row_stride(h) is None):
            h = h.contiguous()
        weight = _kept(weight, shape[-1:], (dtype, torch.float32), device).contiguous()
        inverse = _kept(inverse, shape[:-1], (torch.float32,), device).contiguous()
        dim = shape[-1]
        needs_weight = ctx.needs_input_grad[1]
        grad_y = grad_y.resolve_neg().contiguous()
        grad_h = torch.empty(h.shape, device=device, dtype=h.dtype)
        grad_weight = torch.empty_like(weight) if needs_weight else None
        grad_residual = grad_h if ctx.needs_input_grad[2] else None
        if h.numel() == 0:
            return grad_h, grad_weight.zero_() if needs_weight else None, grad_residual, None
        args = _lib.DsaNormGradArgs()
        args.h, args.inverse, args.weight = h.data_ptr(), inverse.data_ptr(), weight.data_ptr()
        args.grad_out, args.grad_in = grad_y.data_ptr(), grad_h.data_ptr()
        if grad_total is not None:
            grad_total = grad_total.resolve_neg().contiguous()
            args.grad_sum = grad_total.data_ptr()
        args.rows, args.h_stride, args.dim, args.dtype = h.numel() // dim, _row_stride(h), dim, DTYPES[h.dtype]
        args.weight_f32 = weight.dtype == torch.float32
        if needs_weight:
            size = _lib.load().dsa_rms_norm_grad_ws_bytes(args.rows, dim)
            workspace = torch.empty(size, device=device, dtype=torch.uint8)
            args.grad_weight, args.workspace, args.workspace_bytes = grad_weight.data_ptr(), workspace.data_ptr(), size
        _launch("dsa_rms_norm_grad", args, device)
        return grad_h, grad_weight, grad_residual, None


def rms_norm(x, weight, residual=None, *, eps=1e-6):
    """``x [..., dim]`` over its root mean square, times ``weight [dim]``:
    ``h / sqrt(mean(h ** 2) + eps) * weight``, where ``h`` is ``x``, or with a
    ``residual`` the stream ``x + residual``, rounded to its type.

    Returns ``y``, or with a residual ``(y, h)``: new contiguous tensors of ``x``'s
    type.  Sums and products are 32-bit, ``y`` rounded once; a row whose squares leave
    their range, at either end, is multiplied by a power of two first.  A row of zeros
    with ``eps=0``, and one with an infinity or a NaN, are what the formula says.

    ``x`` and ``residual``: bf16, fp16 or fp32, dim up to 16384, evenly spaced rows
    any distance apart (a slice of a projection's output goes in as it is);
    ``weight`` of the same type or fp32.

    Gradients of ``x``, ``residual`` and ``weight`` are recorded where one of them
    requires it (once: there are none of the second order), sums over the rows in
    a fixed order; forward-mode tangents are refused.  In a graph's capture so is a leaf
    whose results of eager calls on the default stream are still kept with their graph:
    its gradient there would end the process, so the call itself says so, whether or not
    a gradient would follow (``torch.no_grad`` captures the norm alone)."""
    fast = _fast_layer()
    if fast is not None:  # checked, allocated and launched in C++ (None: not taken)
        taken = fast.rms_norm(x, weight, residual, eps)
        if taken is not None:
            if type(taken) is int:
                _lib.check(taken, "dsa_rms_norm")
            return taken
    if weight is None:
        raise ValueError("weight must be a tensor")
    _check(x, weight, residual, eps)
    grad, tangent = _derivatives(x, weight, residual)
    if tangent:
        raise ValueError("rms_norm has no forward-mode derivative")
    x, weight, residual = _plain(x, weight, residual)
    if grad:
        if fast is not None:
            fast.capturable(x, weight, residual)
        return _RmsNorm.apply(x, weight, residual, eps)
    y, total, _ = _norm(x, weight, residual, eps, False)
    return y if residual is None else (y, total)


def _codes(x, weight, residual, eps, pow2_scales):
    dim = _check(x, weight, residual, eps)
    if dim % 16:
        raise ValueError(f"codes need a last dimension that is a multiple of 16 (got {dim})")
    if any(_derivatives(x, weight, residual)):
        raise ValueError("codes record no gradient and no forward-mode tangent: call it without them (torch.no_grad)")
    x, weight, residual = _plain(x, weight, residual)
    codes = torch.empty(x.shape, device=x.device, dtype=torch.float8_e4m3fn)
    scales = torch.empty((*x.shape[:-1], -(-dim // SCALE_BLOCK)), device=x.device, dtype=torch.float32)
    total = None if residual is None else torch.empty(x.shape, device=x.device, dtype=x.dtype)
    if x.numel() > 0:
        args = _norm_args(x, weight, residual, eps, codes, total)
        args.scales, args.pow2_scales = scales.data_ptr(), bool(pow2_scales)
        _launch("dsa_rms_norm_fp8", args, x.device)
    return (codes, scales) if residual is None else (codes, scales, total)


def rms_norm_fp8(x, weight, residual=None, *, eps=1e-6, pow2_scales=True):
    """:func:`rms_norm` with 8-bit codes for :func:`dsa_amd.matmul_fp8` in place of
    ``y``: ``codes [..., dim]`` (float8_e4m3fn) and ``scales [..., ceil(dim / 128)]``
    (fp32), which stand for ``codes * scales``, made of the 32-bit ``y``.

    Returns ``(codes, scales)``, or with a residual ``(codes, scales, h)``.  A scale is
    the least power of two that is not below the largest of its 128 values over 448
    (``pow2_scales=False``: that quotient itself); 1 where all are zero.  A block with a
    NaN has a scale of 1 too: a NaN has its own code, and the other values there are coded
    as they are, past 448 as 448 and below 2^-10 as 0.  Without one an infinity makes its
    block's scale infinite: its code is NaN, the others' 0.

    dim: a multiple of 16 up to 16384.  No gradient is recorded, and no input may
    require one while gradients are enabled, or carry a forward-mode tangent."""
    fast = _fast_layer()
    if fast is not None:
        taken = fast.rms_norm_fp8(x, weight, residual, eps, pow2_scales)
        if taken is not None:
            if type(taken) is int:
                _lib.check(taken, "dsa_rms_norm_fp8")
            return taken
    if weight is None:
        raise ValueError("weight must be a tensor")
    return _codes(x, weight, residual, eps, pow2_scales)


def quantize_fp8(x, *, pow2_scales=True):
    """``x [..., dim]`` as 8-bit codes and scales, as :func:`rms_norm_fp8` makes them,
    without a norm: ``(codes, scales)``, for the output of :func:`dsa_amd.forward` or
    :func:`dsa_amd.project_uv` in front of an 8-bit output projection."""
    fast = _fast_layer()
    if fast is not None:
        taken = fast.quantize_fp8(x, pow2_scales)
        if taken is not None:
            if type(taken) is int:
                _lib.check(taken, "dsa_rms_norm_fp8")
            return taken
    return _codes(x, None, None, 0.0, pow2_scales)
