"""Rotary positions for the attention's and the indexer's inputs (no reference
counterpart: the reference takes ``q_rope`` and ``k_rope`` rotated,
README.md:19-21).

:func:`rotary` turns part of each head by its token's position; the cache row
writer (:func:`dsa_amd.write_kv_rows`) does the same to ``k_rope`` on its way
into the cache.  Both take the angles as frequencies (radians a position, one
a pair, 64 bits), which :func:`rotary_frequencies` makes, and form every angle
in 64 bits on the GPU: there is no table of cosines and no largest position.
"""
from __future__ import annotations

import ctypes
import math

import torch

from . import _lib
from .api import _fast_cache, _on_device

ROTARY_MAX_DIM = 512
DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


def rotary_frequencies(dim: int, theta: float = 10000.0, *, scaling=None, factor: float = 1.0,
                       original_length: int = 4096, beta_fast: float = 32.0, beta_slow: float = 1.0, device=None):
    """Frequencies of the ``dim // 2`` pairs, float64: ``theta ** (-2 i / dim)``.

    ``scaling`` stretches them for contexts ``factor`` times ``original_length``:
    ``"linear"`` divides all of them by ``factor``; ``"yarn"`` only those that
    turn fewer than ``beta_slow`` times in ``original_length`` positions, keeps
    those that turn more than ``beta_fast`` times, and goes linearly between the
    two over the pair's number (the borders rounded outward, as published).
    YaRN's factor on the attention scores is the caller's: :func:`rotary`'s
    ``magnitude``, or the softmax scale."""
    if type(dim) is not int or dim < 2 or dim % 2 or dim > ROTARY_MAX_DIM:
        raise ValueError(f"dim must be an even int in [2, {ROTARY_MAX_DIM}]")
    if not (theta > 1.0 and math.isfinite(theta)):
        raise ValueError("theta must be a finite number above 1")
    if scaling not in (None, "linear", "yarn"):
        raise ValueError('scaling must be None, "linear" or "yarn"')
    if not (factor > 0.0 and math.isfinite(factor)):
        raise ValueError("factor must be a positive finite number")
    i = torch.arange(dim // 2, dtype=torch.float64)
    freq = float(theta) ** (-2.0 * i / dim)
    if scaling == "linear":
        freq = freq / factor
    elif scaling == "yarn":
        if not (original_length > 0 and 0.0 < beta_slow < beta_fast):
            raise ValueError("yarn needs original_length > 0 and 0 < beta_slow < beta_fast")

        def pair_of(turns):  # the pair that turns so often in original_length positions
            return dim * math.log(original_length / (turns * 2.0 * math.pi)) / (2.0 * math.log(theta))

        low = max(math.floor(pair_of(beta_fast)), 0)
        high = min(math.ceil(pair_of(beta_slow)), dim - 1)
        stretched = ((i - low) / max(high - low, 0.001)).clamp(0.0, 1.0)
        freq = freq * (1.0 - stretched) + freq / factor * stretched
    return freq.to(device) if device is not None else freq


def check_frequencies(frequencies, device):
    if not isinstance(frequencies, torch.Tensor) or frequencies.dim() != 1 or frequencies.dtype != torch.float64:
        raise ValueError("frequencies must be a 1-D float64 tensor (rotary_frequencies)")
    dim = 2 * frequencies.numel()
    if dim < 2 or dim > ROTARY_MAX_DIM:
        raise ValueError(f"frequencies must hold 1 to {ROTARY_MAX_DIM // 2} values")
    if frequencies.device != device or not frequencies.is_contiguous():
        raise ValueError("frequencies must be contiguous and on the same ROCm GPU as the other inputs")
    return dim


def check_positions(positions, shape, device):
    if not isinstance(positions, torch.Tensor) or positions.shape != shape:
        raise ValueError(f"positions must be {list(shape)}, one for each token")
    if positions.dtype not in (torch.int32, torch.int64):
        raise ValueError("positions must be int32 or int64")
    if positions.device != device or not positions.is_contiguous():
        raise ValueError("positions must be contiguous and on the same ROCm GPU as the other inputs")


def check_magnitude(magnitude):
    if isinstance(magnitude, bool) or not isinstance(magnitude, (int, float)):
        raise TypeError("magnitude must be a float")
    if not abs(magnitude) <= 3.4028234663852886e38:
        raise ValueError("magnitude must be a finite 32-bit number")


def written(t):
    """Tells autograd of a tensor that a call has written in place."""
    if not t.is_inference():
        torch.autograd.graph.increment_version(t)


def _span(t):
    """Addresses [first, last) that the tensor's elements lie in."""
    last = sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1
    return t.data_ptr(), t.data_ptr() + last * t.element_size()


def _elements_distinct(t):
    """Whether no two elements share memory: each dimension steps over the ones inside it."""
    reach = 1
    for s, n in sorted((s, n) for n, s in zip(t.shape, t.stride()) if n > 1):
        if s < reach:
            return False
        reach += (n - 1) * s
    return True


def has_tangent(t):
    """Whether the tensor carries a forward-mode derivative."""
    return torch.autograd.forward_ad.unpack_dual(t).tangent is not None


class _Rotary(torch.autograd.Function):
    """Linear in x: the tangent takes the same turn, the gradient the opposite one."""

    @staticmethod
    def forward(ctx, x, positions, frequencies, interleaved, start, transposed, magnitude):
        ctx.save_for_backward(positions, frequencies)
        ctx.save_for_forward(positions, frequencies)
        ctx.how = (interleaved, start, transposed, magnitude)
        return _launch(x, positions, frequencies, interleaved, start, transposed, magnitude,
                       torch.empty(x.shape, device=x.device, dtype=x.dtype))

    @staticmethod
    def _turned(ctx, t, back):
        return rotary(t if t.stride(-1) == 1 else t.contiguous(), *ctx.saved_tensors, interleaved=ctx.how[0],
                      start=ctx.how[1], transposed=bool(ctx.how[2]) != back, magnitude=ctx.how[3])

    @staticmethod
    def backward(ctx, grad):
        return _Rotary._turned(ctx, grad, True), None, None, None, None, None, None

    @staticmethod
    def jvp(ctx, tangent, *_):
        return _Rotary._turned(ctx, tangent, False)


def rotary(x, positions, frequencies, *, interleaved=True, start=0, transposed=False, magnitude=1.0, out=None):
    """``x [..., H, D]`` with the pairs of ``x[..., start:start + dim]`` turned by
    ``positions * frequencies`` (``dim = 2 * len(frequencies)``).

    Pair ``i`` is the elements ``2 i, 2 i + 1`` of the rotated part
    (``interleaved``; attention heads) or ``i, i + dim / 2`` (half layout; the
    indexer's heads): ``y0 = magnitude (x0 cos - x1 sin)``, ``y1 = magnitude
    (x0 sin + x1 cos)``.  The rest of each head is copied.

    ``x``: ``[tokens, H, D]`` or ``[B, SQ, H, D]``, bf16, fp16 or fp32, any strides but a last
    one of 1, so a slice of a projection's output goes in as it is
    (``rotary(q[..., 128:], ...)`` gives :func:`dsa_amd.forward`'s ``q_rope``);
    ``positions`` int32 or int64, ``x.shape[:-2]``; ``frequencies`` float64.
    The products are 32-bit and rounded once.

    ``out``: where the result goes (``x`` itself: in place, the rest of each head
    untouched), else a new contiguous tensor.  ``transposed`` turns the other
    way, which is the gradient for ``x``; where ``x`` requires a gradient or
    carries a forward-mode tangent the call records that itself (not with ``out``).
    There is no gradient for ``frequencies``, and none may be asked of them."""
    fast = _fast_cache()
    if fast is not None:  # checked and launched in C++ (None: not taken)
        taken = fast.rotary(x, positions, frequencies, interleaved, start, transposed, magnitude, out)
        if taken is not None:
            if type(taken) is int:
                _lib.check(taken, "dsa_rotary")
            return taken
    if not isinstance(x, torch.Tensor) or x.dim() not in (3, 4):
        raise ValueError("x must be [tokens, H, D] or [B, SQ, H, D]")
    device = x.device
    if device.type != "cuda" or torch.version.hip is None:
        raise ValueError("x must be on a ROCm GPU")
    if x.dtype not in DTYPES:
        raise ValueError("x must be bfloat16, float16 or float32")
    dim = check_frequencies(frequencies, device)
    if (torch.is_grad_enabled() and frequencies.requires_grad) or has_tangent(frequencies):
        raise ValueError("frequencies must not require a gradient: there is none for them")
    check_positions(positions, x.shape[:-2], device)
    check_magnitude(magnitude)
    if type(start) is not int or start < 0 or start + dim > x.shape[-1]:
        raise ValueError(f"start must be an int with start + {dim} inside the head of {x.shape[-1]}")
    if x.stride(-1) != 1:
        raise ValueError("x's last stride must be 1")
    wants_grad = (torch.is_grad_enabled() and x.requires_grad) or has_tangent(x)
    if out is not None:
        if not isinstance(out, torch.Tensor) or out.shape != x.shape or out.dtype != x.dtype or out.device != device:
            raise ValueError("out must have x's shape, type and device")
        if out.stride(-1) != 1 or not _elements_distinct(out):
            raise ValueError("out's last stride must be 1 and no two of its elements share memory")
        if wants_grad or (torch.is_grad_enabled() and out.requires_grad) or has_tangent(out):
            raise ValueError("out cannot be given where a gradient is recorded")
        same = out.data_ptr() == x.data_ptr() and out.stride() == x.stride()
        if not same and x.numel() > 0:
            (x0, x1), (y0, y1) = _span(x), _span(out)
            if x0 < y1 and y0 < x1:
                raise ValueError("out must be x itself or lie apart from it")
        written(out)
    elif wants_grad:
        return _Rotary.apply(x, positions, frequencies, interleaved, start, transposed, magnitude)
    else:
        out = torch.empty(x.shape, device=device, dtype=x.dtype)
    return _launch(x, positions, frequencies, interleaved, start, transposed, magnitude, out)


def _launch(x, positions, frequencies, interleaved, start, transposed, magnitude, out):
    if x.numel() == 0:
        return out
    args = _lib.DsaRotaryArgs()
    args.x, args.out, args.positions = x.data_ptr(), out.data_ptr(), positions.data_ptr()
    args.frequencies = frequencies.data_ptr()
    groups = x.shape[0] if x.dim() == 4 else 1
    tokens, heads, width = x.shape[-3:]
    args.groups, args.tokens = groups, tokens
    xs, ys = x.stride(), out.stride()
    args.x_stride[:] = (xs[0] if x.dim() == 4 else 0, xs[-3], xs[-2])
    args.out_stride[:] = (ys[0] if x.dim() == 4 else 0, ys[-3], ys[-2])
    args.heads, args.width, args.start, args.dim = heads, width, start, 2 * frequencies.numel()
    args.dtype = DTYPES[x.dtype]
    args.positions_64 = positions.dtype == torch.int64
    args.interleaved, args.transposed, args.magnitude = bool(interleaved), bool(transposed), magnitude
    device = x.device
    with _on_device(device):
        rc = _lib.load().dsa_rotary(ctypes.byref(args), torch._C._cuda_getCurrentRawStream(device.index))
    if rc:
        _lib.check(rc, "dsa_rotary")
    return out
