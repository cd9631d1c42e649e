"""The paged kv cache from step to step: blocks for new tokens, and their rows
(no reference counterpart: the reference takes a contiguous cache as given,
dsa/api.py:30-33).

A serving step runs :func:`extend_block_table` (blocks, slots and positions of
its new tokens, from the requests' lengths, on the GPU),
:func:`dsa_amd.rotary` on its queries, :func:`write_kv_rows` on its new rows,
and then :func:`dsa_amd.forward` (or :func:`dsa_amd.forward_shared`) with the
block table.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from .api import FP8_ROW, HEAD_DIM, ROPE_DIM, _fast_cache, _on_device
from .rotary import check_frequencies, check_magnitude, check_positions, has_tangent, written

MAX_SEQUENCES = 4096


def _int32_vector(t, name, device, size=None):
    if not isinstance(t, torch.Tensor) or t.dim() != 1 or (size is not None and t.shape[0] != size):
        raise ValueError(f"{name} must be [{'n' if size is None else size}]")
    if t.dtype != torch.int32:
        raise ValueError(f"{name} must be int32")
    if t.device != device or not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous and on the same ROCm GPU as the other inputs")


def extend_block_table(block_table, lengths, new_tokens, free_blocks, block_size: int, max_tokens: int):
    """One step's blocks and slots: sequence ``b`` holds ``lengths[b]`` tokens and
    gets ``new_tokens[b]`` more.

    ``block_table`` int32 ``[B, max_blocks]`` is updated in place: the
    ``ceil((lengths + new_tokens) / block_size) - ceil(lengths / block_size)``
    blocks that a sequence still needs are taken from the front of
    ``free_blocks`` (int32 ``[n]``), the first sequence's first.  No other entry
    is touched, so whole blocks that sequences share stay shared.

    Returns int32 tensors ``(slots, positions, starts, totals, used)``:

    * ``slots [max_tokens]``: the cache row of each new token, sequence after
      sequence (the ``slots`` of :func:`write_kv_rows`); -1 behind the last
      one, and where the list was short, the row too narrow, or the entry of a
      partly filled block negative;
    * ``positions [max_tokens]``: each one's position (``positions + 1`` is the
      number of keys it sees); 0 behind the last one;
    * ``starts [B + 1]``: the first token of each sequence, and their number
      (tokens from ``max_tokens`` on are left out of ``slots`` and ``positions``);
    * ``totals [B]``: ``lengths + new_tokens``;
    * ``used [1]``: blocks taken; above ``len(free_blocks)`` the list was short.

    One launch, nothing synchronised, B up to 4096."""
    fast = _fast_cache()
    if fast is not None:  # checked and launched in C++ (None: not taken)
        taken = fast.extend_block_table(block_table, lengths, new_tokens, free_blocks, block_size, max_tokens)
        if taken is not None:
            if type(taken) is int:
                _lib.check(taken, "dsa_extend_block_table")
            return taken
    if not isinstance(block_table, torch.Tensor) or block_table.dim() != 2 or min(block_table.shape) <= 0:
        raise ValueError("block_table must be [B, max_blocks]")
    if type(block_size) is not int or not 0 < block_size < 2 ** 31:
        raise ValueError("block_size must be a positive int")
    if type(max_tokens) is not int or not 0 <= max_tokens < 2 ** 31:
        raise ValueError("max_tokens must be an int, not negative")
    batch, max_blocks = block_table.shape
    if batch > MAX_SEQUENCES:
        raise ValueError(f"at most {MAX_SEQUENCES} sequences (got {batch})")
    device = block_table.device
    if device.type != "cuda" or torch.version.hip is None or not block_table.is_contiguous():
        raise ValueError("block_table must be contiguous on a ROCm GPU")
    if block_table.dtype != torch.int32:
        raise ValueError("block_table must be int32")
    _int32_vector(lengths, "lengths", device, batch)
    _int32_vector(new_tokens, "new_tokens", device, batch)
    _int32_vector(free_blocks, "free_blocks", device)
    out = torch.empty(2 * max_tokens + 2 * batch + 2, device=device, dtype=torch.int32)
    slots, positions, starts, totals, used = out.split([max_tokens, max_tokens, batch + 1, batch, 1])
    with _on_device(device):
        rc = _lib.load().dsa_extend_block_table(
            block_table.data_ptr(), lengths.data_ptr(), new_tokens.data_ptr(), free_blocks.data_ptr(), slots.data_ptr(),
            positions.data_ptr(), starts.data_ptr(), totals.data_ptr(), used.data_ptr(), batch, max_blocks, block_size,
            free_blocks.numel(), max_tokens, torch._C._cuda_getCurrentRawStream(device.index))
    if rc:
        _lib.check(rc, "dsa_extend_block_table")
    written(block_table)
    return slots, positions, starts, totals, used


def write_kv_rows(kv, k_rope, slots, kv_cache, rope_cache=None, *, positions=None, frequencies=None, interleaved=True,
                  magnitude=1.0, pow2_scales=True):
    """New tokens' rows into a cache, in place: row ``slots[i]`` of the cache
    becomes token ``i``'s ``kv`` and ``k_rope``.

    ``kv [tokens, 512]`` and ``k_rope [tokens, 64]`` bf16, each row contiguous and
    any distance apart (so the two slices of a projection's output go in as they
    are); ``slots`` int32 ``[tokens]``, rows of the cache with its leading
    dimensions flattened.  A token whose slot lies outside the cache is left out.
    No row may be named twice: nothing orders the two tokens' writes, and the row
    holds parts of either (as :func:`extend_block_table` gives them, slots are
    distinct).  ``kv`` and ``k_rope`` may be rows of the cache themselves, but not
    ones that the call writes.

    ``kv_cache``: a bf16 cache or pool ``[..., 512]`` with its ``rope_cache
    [..., 64]``, or an fp8 one, uint8 ``[..., 656]``, whose rows become those of
    :func:`dsa_amd.quantize_kv_fp8` (``pow2_scales`` as there).

    No gradient is recorded and no forward-mode tangent, and the caches must not
    require the one or carry the other.

    ``frequencies`` (float64 ``[32]``) with ``positions`` (int32 or int64
    ``[tokens]``) turns ``k_rope`` on its way as :func:`dsa_amd.rotary` does."""
    fast = _fast_cache()
    if fast is not None:  # checked and launched in C++ (None: not taken)
        rc = fast.write_kv_rows(kv, k_rope, slots, kv_cache, rope_cache, positions, frequencies, interleaved, magnitude,
                                pow2_scales)
        if rc is not None:
            if rc:
                _lib.check(rc, "dsa_write_kv_rows")
            return
    if (not isinstance(kv, torch.Tensor) or not isinstance(k_rope, torch.Tensor) or kv.dim() != 2 or k_rope.dim() != 2
            or kv.shape[1] != HEAD_DIM or k_rope.shape != (kv.shape[0], ROPE_DIM)):
        raise ValueError("expected kv[tokens, 512] and k_rope[tokens, 64]")
    if not isinstance(kv_cache, torch.Tensor):
        raise ValueError("kv_cache must be a tensor")
    device = kv.device
    fp8 = kv_cache.dtype == torch.uint8
    if fp8 and rope_cache is not None:
        raise ValueError("with an fp8 kv_cache rope_cache must be None: the rope values are in the rows")
    if not fp8 and not isinstance(rope_cache, torch.Tensor):
        raise ValueError("rope_cache is required unless kv_cache holds fp8 rows (uint8 [..., 656])")
    if kv_cache.dim() < 2 or kv_cache.shape[-1] != (FP8_ROW if fp8 else HEAD_DIM) or (
            not fp8 and rope_cache.shape != (*kv_cache.shape[:-1], ROPE_DIM)):
        raise ValueError("expected kv_cache[..., 512] and rope_cache[..., 64] of the same leading dims, "
                         "or kv_cache uint8[..., 656]")
    if (device.type != "cuda" or torch.version.hip is None or k_rope.device != device or kv_cache.device != device
            or not kv_cache.is_contiguous()
            or (not fp8 and (rope_cache.device != device or not rope_cache.is_contiguous()))):
        raise ValueError("all tensors must be on the same ROCm GPU and the caches contiguous")
    bf16 = torch.bfloat16
    if kv.dtype != bf16 or k_rope.dtype != bf16 or (not fp8 and (kv_cache.dtype != bf16 or rope_cache.dtype != bf16)):
        raise ValueError("kv, k_rope and a cache that is not uint8 must be bfloat16")
    tokens = kv.shape[0]
    if (kv.stride(1) != 1 or k_rope.stride(1) != 1
            or (tokens > 1 and (kv.stride(0) % 8 or k_rope.stride(0) % 2))
            or kv.data_ptr() % 16 or k_rope.data_ptr() % 4 or kv_cache.data_ptr() % 16
            or (not fp8 and rope_cache.data_ptr() % 4)):
        raise ValueError("kv needs contiguous rows, 16-byte aligned and a multiple of 8 elements apart, k_rope rows "
                         "4-byte aligned and a multiple of 2 apart; the caches must be 16- and 4-byte aligned")
    if not fp8 and any((torch.is_grad_enabled() and t.requires_grad) or has_tangent(t) for t in (kv_cache, rope_cache)):
        raise ValueError("the caches are written in place and must not require a gradient")
    _int32_vector(slots, "slots", device, tokens)
    if (frequencies is None) != (positions is None):
        raise ValueError("positions and frequencies go together")
    if frequencies is not None:
        if check_frequencies(frequencies, device) != ROPE_DIM:
            raise ValueError("frequencies must hold 32 values")
        check_positions(positions, kv.shape[:1], device)
    check_magnitude(magnitude)
    rows = kv_cache.numel() // kv_cache.shape[-1]
    if tokens == 0 or rows == 0:
        return
    args = _lib.DsaWriteArgs()
    args.kv, args.k_rope, args.slots = kv.data_ptr(), k_rope.data_ptr(), slots.data_ptr()
    args.cache, args.rope_cache = kv_cache.data_ptr(), None if fp8 else rope_cache.data_ptr()
    if frequencies is not None:
        args.positions, args.frequencies = positions.data_ptr(), frequencies.data_ptr()
        args.positions_64 = positions.dtype == torch.int64
    args.tokens, args.cache_rows = tokens, rows
    args.kv_stride, args.rope_stride = (kv.stride(0), k_rope.stride(0)) if tokens > 1 else (HEAD_DIM, ROPE_DIM)
    args.kv_format = _lib.KV_FP8 if fp8 else _lib.KV_BF16
    args.pow2_scales, args.interleaved, args.magnitude = bool(pow2_scales), bool(interleaved), magnitude
    with _on_device(device):
        rc = _lib.load().dsa_write_kv_rows(ctypes.byref(args), torch._C._cuda_getCurrentRawStream(device.index))
    if rc:
        _lib.check(rc, "dsa_write_kv_rows")
    written(kv_cache)
    if not fp8:
        written(rope_cache)
