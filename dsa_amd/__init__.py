"""MI355X-native DSA sparse-MLA attention forward (drop-in for ``dsa.forward``).

Public surface mirrors the reference package (dsa/__init__.py:2-5):
``forward``, ``Tuning``, ``CASE_SHAPES``, ``SELECTED``; plus ``merge`` (the
standalone FP32 split merge), ``select`` (the plan for a shape) and the
lightning indexer that produces the indices (``indexer``, ``indexer_logits``,
``indexer_topk``), the fp8 kv cache row writer (``quantize_kv_fp8``) and the
W_UV output projection after the attention (``project_uv``, ``merge_uv``,
``forward(w_uv=)``) and the row-range bucketing of prefill-sized calls'
indices (``bucket_indices``); and what a paged cache takes from step to step:
block tables and slot maps from lengths (``extend_block_table``), rotary
positions (``rotary``, ``rotary_frequencies``), cache row writes
(``write_kv_rows``) and dense attention of a batch that shares a prefix
(``forward_shared``); trees of drafted tokens and their attention
(``draft_tree``, ``forward_tree``); and the norms, 8-bit codes and 8-bit products
around the attention (``rms_norm``, ``rms_norm_fp8``, ``quantize_fp8``,
``matmul_fp8``).
"""
from .api import bucket_indices, forward, merge, merge_uv, plan_call, project_uv
from .config import CASE_SHAPES, SELECTED, Tuning, select
from .indexer import indexer, indexer_logits, indexer_topk
from .kvcache import quantize_kv_fp8
from .norm import quantize_fp8, rms_norm, rms_norm_fp8
from .paging import extend_block_table, write_kv_rows
from .product import matmul_fp8
from .rotary import rotary, rotary_frequencies
from .shared import forward_shared, forward_tree
from .tree import draft_tree

__all__ = ["forward", "merge", "merge_uv", "project_uv", "plan_call", "bucket_indices", "Tuning", "CASE_SHAPES",
           "SELECTED", "select", "indexer", "indexer_logits", "indexer_topk", "quantize_kv_fp8", "extend_block_table",
           "write_kv_rows", "rotary", "rotary_frequencies", "forward_shared", "forward_tree", "draft_tree",
           "rms_norm", "rms_norm_fp8", "quantize_fp8", "matmul_fp8"]
