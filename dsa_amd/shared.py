"""Dense MLA attention of a batch that shares a prefix (no reference
counterpart: the reference attends to given indices, dsa/api.py:76-132).

Beside :func:`dsa_amd.forward`, over the same caches: contexts shorter than the
indexer's top-k, a model's dense layers, and batches whose sequences start with
the same rows -- a system prompt, a document -- which are then read, and their
products formed, once for the whole batch (``csrc/shared_attn.hip``); and steps
that verify a tree of drafted tokens behind each sequence.  There is no CPU path.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from .api import FP8_ROW, HEAD_DIM, ROPE_DIM, _check_scale, _device_cus, _fast_cache, _on_device
from .tree import TREE_MAX_WORDS


def _check(q, kv, q_rope, k_rope, lengths, prefix, block_table, tree=None):
    optional = [t for t in (k_rope, block_table, tree) if t is not None]
    if not all(isinstance(t, torch.Tensor) for t in (q, kv, q_rope, lengths, *optional)):
        raise ValueError("q, kv, q_rope, lengths (and k_rope, block_table) must be tensors")
    fp8 = kv.dtype == torch.uint8
    if fp8 and k_rope is not None:
        raise ValueError("with fp8 kv rows (uint8 [..., 656]) k_rope must be None: the rope values are in the rows")
    if not fp8 and k_rope is None:
        raise ValueError("k_rope is required unless kv holds fp8 rows (uint8 [..., 656])")
    if q.dim() != 4 or kv.dim() != 4:
        raise ValueError("q and kv must be 4-D tensors")
    batch, queries, heads, width = q.shape
    if tree is not None and (tree.dim() != 3 or tree.shape[:2] != (batch, queries)
                             or not 1 <= tree.shape[2] <= TREE_MAX_WORDS):
        raise ValueError(f"tree must be [B, SQ, words] of up to {TREE_MAX_WORDS} words (draft_tree)")
    if tree is not None and lengths.shape != (batch,):
        raise ValueError("with a tree lengths must be [B]")
    if block_table is None:
        pool, length = (batch, kv.shape[1]), kv.shape[1]
    else:
        if block_table.dim() != 2 or block_table.shape[0] != batch:
            raise ValueError("block_table must be [B, max_blocks]")
        pool, length = tuple(kv.shape[:2]), block_table.shape[1] * kv.shape[1]
    if (width != HEAD_DIM or kv.shape != (*pool, 1, FP8_ROW if fp8 else HEAD_DIM)
            or q_rope.shape != (batch, queries, heads, ROPE_DIM)
            or (not fp8 and k_rope.shape != (*pool, 1, ROPE_DIM)) or (tree is None and lengths.shape != (batch, queries))
            or min(batch, queries, heads, length, *pool) <= 0):
        raise ValueError("expected q[B,SQ,H,512], q_rope[B,SQ,H,64], lengths[B,SQ], kv[B,L,1,512] and k_rope[B,L,1,64] "
                         "or fp8 kv[B,L,1,656] (or pools [N,BS,1,...] with block_table[B,M])")
    if heads % 16:
        raise ValueError(f"the number of heads must be a multiple of 16 (got {heads})")
    if type(prefix) is not int or not 0 <= prefix <= length:
        raise ValueError(f"prefix must be an int in [0, {length}]")
    device = q.device
    tensors = [q, kv, q_rope, lengths] + ([] if fp8 else [k_rope]) + ([] if block_table is None else [block_table])
    tensors += [] if tree is None else [tree]
    if device.type != "cuda" or torch.version.hip is None or any(
            t.device != device or not t.is_contiguous() for t in tensors):
        raise ValueError("all inputs must be contiguous and on the same ROCm GPU")
    bf16 = torch.bfloat16
    if (q.dtype != bf16 or q_rope.dtype != bf16 or (not fp8 and (kv.dtype != bf16 or k_rope.dtype != bf16))
            or any(t is not None and t.dtype != torch.int32 for t in (lengths, block_table, tree))):
        raise ValueError("q/kv/q_rope/k_rope must be bfloat16, lengths (and block_table, tree) int32")
    return batch, queries, heads, length, device, fp8


def forward_shared(q, kv, q_rope, k_rope, lengths, prefix=0, *, scale=None, block_table=None):
    """Dense MLA attention over the first ``lengths`` rows of each query's sequence,
    of which the first ``prefix`` are the same for the whole batch.

    Returns ``(output, softmax_max, softmax_sum)`` as :func:`dsa_amd.forward`
    does: bf16 ``[B,SQ,H,512]`` and two fp32 ``[B,1,SQ,H]`` (max and sum of
    exp(score - max), not LSE).  ``q``, ``q_rope``, ``kv``, ``k_rope``, ``scale``
    and ``block_table`` as there, contiguous or paged, bf16 or fp8 rows.

    ``lengths`` (int32 ``[B, SQ]``, as the indexer's): query ``t`` of sequence
    ``b`` sees rows ``[0, lengths[b, t])``, clamped to ``[0, L]``; a causal step
    gives each query its position plus one.  A query that sees none (padding)
    gives output 0, max -inf and sum 0.  Rows a query does not see may hold
    anything, infinities and NaN included.  In rows that it sees they do what the
    formulas say: a score of +inf or NaN, or no score above -inf, makes its output
    and sum NaN (max too, where a score is NaN and none +inf); beside finite scores,
    one of -inf is a weight of 0, and 0 times an infinite latent value NaN in that
    value's column.

    ``prefix``: rows ``[0, prefix)`` are read from sequence 0's cache (or through
    its block table row) for every sequence.  The caller vouches that they are
    the same; it need not be a multiple of the block size.  0: nothing shared.

    Scores, sums and statistics are 32-bit; the weights are rounded to bf16, by half a
    step (2^-8 of each) at most, before their product with the values.  The output is
    finite for max|kv| < 2^38.  Caches hold fewer than 2^25 rows.
    Outputs are fresh tensors, which record no gradient and no forward-mode tangent
    (as :func:`dsa_amd.forward`'s), the workspace is the caching allocator's, and
    nothing synchronises."""
    fast = _fast_cache()
    if fast is not None:  # checked, allocated and launched in C++ (None: not taken)
        taken = fast.forward_shared(q, kv, q_rope, k_rope, lengths, prefix, scale, block_table)
        if taken is not None:
            if type(taken) is int:
                _lib.check(taken, "dsa_fwd_shared")
            return taken
    return _run(q, kv, q_rope, k_rope, lengths, None, prefix, scale, block_table)


def forward_tree(q, kv, q_rope, k_rope, lengths, tree, prefix=0, *, scale=None, block_table=None):
    """:func:`forward_shared` for a step that verifies drafted tokens: query ``t`` of
    sequence ``b`` sees rows ``[0, lengths[b])`` and, of the rows behind them, those
    that its words of ``tree`` name -- row ``lengths[b] + j`` where bit ``j % 32`` of
    ``tree[b, t, j // 32]`` is set (:func:`dsa_amd.draft_tree`: the token itself and
    its ancestors).

    ``lengths`` int32 ``[B]``, clamped to ``[0, L]``; ``tree`` int32 ``[B, SQ, words]``,
    up to 64 words, any bits (bits of rows from ``L`` on are left out).  The drafted
    tokens' rows have to be in the cache: token ``j``'s at row ``lengths[b] + j``
    (:func:`dsa_amd.write_kv_rows`), rotated by its own position.  A query with no row
    gives output 0, max -inf and sum 0.

    All else, and the three results, as :func:`forward_shared`'s, its weights in bf16
    among it; rows below ``prefix`` are sequence 0's.  A padding token of
    :func:`dsa_amd.draft_tree` has no bits, and sees its sequence's rows all the same."""
    fast = _fast_cache()
    if fast is not None:  # checked, allocated and launched in C++ (None: not taken)
        taken = fast.forward_tree(q, kv, q_rope, k_rope, lengths, tree, prefix, scale, block_table)
        if taken is not None:
            if type(taken) is int:
                _lib.check(taken, "dsa_fwd_tree")
            return taken
    if not isinstance(tree, torch.Tensor):
        raise ValueError("tree must be a tensor")
    return _run(q, kv, q_rope, k_rope, lengths, tree, prefix, scale, block_table)


def _run(q, kv, q_rope, k_rope, lengths, tree, prefix, scale, block_table):
    scale = _check_scale(scale)
    batch, queries, heads, length, device, fp8 = _check(q, kv, q_rope, k_rope, lengths, prefix, block_table,
                                                          tree)
    call = "dsa_fwd_shared" if tree is None else "dsa_fwd_tree"
    whole = _lib.DsaTreeArgs()
    args = whole.shared
    args.B, args.SQ, args.H, args.L, args.prefix = batch, queries, heads, length, prefix
    args.num_cus = _device_cus(device)
    lib = _lib.load()
    size = lib.dsa_fwd_shared_ws_bytes(ctypes.byref(args))
    if size < 0:
        _lib.check(-1, call)
    output = torch.empty_like(q)
    maximum = torch.empty((batch, 1, queries, heads), device=device, dtype=torch.float32)
    denominator = torch.empty_like(maximum)
    workspace = torch.empty(size, device=device, dtype=torch.uint8)
    args.q, args.kv, args.q_rope, args.lengths = q.data_ptr(), kv.data_ptr(), q_rope.data_ptr(), lengths.data_ptr()
    args.k_rope = None if fp8 else k_rope.data_ptr()
    args.out, args.out_max, args.out_sum = output.data_ptr(), maximum.data_ptr(), denominator.data_ptr()
    args.workspace, args.workspace_bytes = workspace.data_ptr(), size
    args.kv_format = _lib.KV_FP8 if fp8 else _lib.KV_BF16
    args.scale = 0.0 if scale is None else scale
    if block_table is not None:
        args.block_table, args.max_blocks = block_table.data_ptr(), block_table.shape[1]
        args.block_size, args.num_blocks = kv.shape[1], kv.shape[0]
    if tree is not None:
        whole.tree, whole.words = tree.data_ptr(), tree.shape[2]
    with _on_device(device):
        stream = torch._C._cuda_getCurrentRawStream(device.index)
        rc = getattr(lib, call)(ctypes.byref(args if tree is None else whole), stream)
    if rc:
        _lib.check(rc, call)
    return output, maximum, denominator
