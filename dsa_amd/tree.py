"""Trees of drafted tokens (no reference counterpart: the reference attends to
given indices, dsa/api.py:76-132).

A step that verifies drafted tokens gives each of them the rows of its sequence
and, behind those, of its own ancestors: :func:`draft_tree` finds these and the
positions, from each token's parent, and :func:`dsa_amd.forward_tree` attends.
"""
from __future__ import annotations

import torch

from . import _lib
from .api import _fast_cache, _on_device

TREE_MAX_WORDS = 64


def draft_tree(parents, lengths):
    """``(tree, positions)`` of drafted tokens, ``SQ`` behind each of ``B`` sequences.

    ``parents`` int32 ``[B, SQ]``: the number of the drafted token that each follows,
    below its own, or -1 for the sequence's last row.  Anything else, or an ancestor
    with one, makes it padding.  ``lengths`` int32 ``[B]``: rows that each sequence has.

    * ``tree`` int32 ``[B, SQ, ceil(SQ / 32)]``, for :func:`dsa_amd.forward_tree`: bit
      ``j % 32`` of word ``j // 32`` is set where token ``j`` is ``t`` or an ancestor of
      it; none for padding;
    * ``positions`` int32 ``[B, SQ]``: the length plus the number of ancestors (the
      positions for :func:`dsa_amd.rotary`; the token's row stays ``lengths + t``); 0
      for padding.

    One launch, nothing synchronised, SQ up to 2048, B up to 2^20."""
    fast = _fast_cache()
    if fast is not None:  # checked, allocated and launched in C++ (None: not taken)
        taken = fast.draft_tree(parents, lengths)
        if taken is not None:
            if type(taken) is int:
                _lib.check(taken, "dsa_draft_tree")
            return taken
    if not isinstance(parents, torch.Tensor) or parents.dim() != 2 or min(parents.shape) <= 0:
        raise ValueError("parents must be [B, SQ]")
    batch, tokens = parents.shape
    if tokens > 32 * TREE_MAX_WORDS or batch > 1 << 20:
        raise ValueError(f"at most {32 * TREE_MAX_WORDS} tokens behind each of 2^20 sequences (got {tokens}, {batch})")
    if not isinstance(lengths, torch.Tensor) or lengths.shape != (batch,):
        raise ValueError("lengths must be [B]")
    device = parents.device
    if device.type != "cuda" or torch.version.hip is None or lengths.device != device or not (
            parents.is_contiguous() and lengths.is_contiguous()):
        raise ValueError("all inputs must be contiguous and on the same ROCm GPU")
    if parents.dtype != torch.int32 or lengths.dtype != torch.int32:
        raise ValueError("parents and lengths must be int32")
    tree = torch.empty((batch, tokens, -(-tokens // 32)), device=device, dtype=torch.int32)
    positions = torch.empty_like(parents)
    with _on_device(device):
        rc = _lib.load().dsa_draft_tree(parents.data_ptr(), lengths.data_ptr(), tree.data_ptr(), positions.data_ptr(),
                                        batch, tokens, torch._C._cuda_getCurrentRawStream(device.index))
    if rc:
        _lib.check(rc, "dsa_draft_tree")
    return tree, positions
